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
constexpr float LP_LOG2E = 1.4426950408889634f, LP_LN2 = 0.69314718055994531f;

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

__device__ __forceinline__ float exp2_approx(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

constexpr float LP_LOWEST = -3.402823466e38f;
// What the logarithm of a probability (by any base) counts as at least where it is multiplied by that probability, which is 0 in fp32 from
// -150 on: 0, not NaN, for -inf.  It is bounded behind the multiplication by the scale, which may be as small as fp32 has it.
constexpr float LP_NOTHING = -1e4f;
// s / ln 2, finite for every scale.
__device__ __forceinline__ float lp_factor(float scale) { return fminf(scale * LP_LOG2E, -LP_LOWEST); }

__device__ __forceinline__ long long lp_token(const void* tokens, int wide, long long row) {
  return wide ? reinterpret_cast<const long long*>(tokens)[row] : (long long)reinterpret_cast<const int*>(tokens)[row];
}

// Largest logit so far (NaN left out: it shows in the sum), sum = S and with c = s / ln 2 dist = sum 2^(c (x - top)) c (x - top).  Of
// nothing: the lowest number, which no -inf reaches, and zeros.
struct RowSums {
  float top, sum, dist;
};
// And the largest logits of a thread's even and odd packs.
struct ShareSums {
  RowSums r;
  float top_a, top_b;
};
// The same, seen from `top`, which is not below its own.
__device__ __forceinline__ void lp_raise(RowSums& r, float top, float c) {
  const float a = fmaxf((r.top - top) * c, LP_NOTHING), f = exp2_approx(a);
  r.dist = fmaf(r.sum, a, r.dist) * f;
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
      float a0, a1;
      unpack_f32x2(mul_f32x2(sub_f32x2(pack_f32x2(x[i], x[i + 1]), top2), c2), a0, a1);
      a0 = max_nan(a0, LP_NOTHING);
      a1 = max_nan(a1, LP_NOTHING);
      const unsigned long long e2 = pack_f32x2(exp2_approx(a0), exp2_approx(a1));
      sum2 = add_f32x2(sum2, e2);
      fma_f32x2(dist2, e2, pack_f32x2(a0, a1));
    }
    float s0, s1, d0, d1;
    unpack_f32x2(sum2, s0, s1);
    unpack_f32x2(dist2, d0, d1);
    r.sum += s0 + s1;
    r.dist += d0 + d1;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float a = max_nan((x[i] - r.top) * c, LP_NOTHING), e = exp2_approx(a);
      r.sum += e;
      r.dist = fmaf(e, a, r.dist);
    }
  }
}

// What a row's sums give: the logarithm of S and the entropy; a row of nothing has the sum 0.
__device__ __forceinline__ void lp_finish(const LogProbArgs& g, long long row, const RowSums& r, float log_sum, float token_logit, long long token) {
  const bool empty = r.sum == 0.f;
  if (g.out)
    g.out[row] = token < 0 || token >= g.mask_cols ? 0.f : token >= g.cols || empty ? -INFINITY : g.scale * (token_logit - r.top) - log_sum;
  if (g.entropy) g.entropy[row] = empty ? 0.f : log_sum - LP_LN2 * (r.dist / r.sum);
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
  const float c = lp_factor(g.scale);
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

// The largest of a pack's logits, NaN left out.
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
// What a logit counts as at least in the fast sums, so that no product of them is 0 times infinity: -2^100, in f16 the lowest number.
template <typename T>
__device__ __forceinline__ float lp_low() { return std::is_same<T, __half>::value ? -65504.f : -1.2676506002282294e30f; }
template <typename T>
__device__ __forceinline__ void lp_lift(SbWords<16>& w);
template <>
__device__ __forceinline__ void lp_lift<float>(SbWords<16>& w) {
  const float low = lp_low<float>();
  w.v.x = __float_as_uint(max_nan(__uint_as_float(w.v.x), low));
  w.v.y = __float_as_uint(max_nan(__uint_as_float(w.v.y), low));
  w.v.z = __float_as_uint(max_nan(__uint_as_float(w.v.z), low));
  w.v.w = __float_as_uint(max_nan(__uint_as_float(w.v.w), low));
}
template <>
__device__ __forceinline__ void lp_lift<__nv_bfloat16>(SbWords<16>& w) {
  const __nv_bfloat162 low = __float2bfloat162_rn(lp_low<__nv_bfloat16>());
  __nv_bfloat162 v[4];
  memcpy(v, &w, 16);
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = __hmax2_nan(v[i], low);
  memcpy(&w, v, 16);
}
template <>
__device__ __forceinline__ void lp_lift<__half>(SbWords<16>& w) {
  const __half2 low = __float2half2_rn(lp_low<__half>());
  __half2 v[4];
  memcpy(v, &w, 16);
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = __hmax2_nan(v[i], low);
  memcpy(&w, v, 16);
}

// The pairs of a pack as fp32.
template <typename T>
__device__ __forceinline__ void lp_pairs(const SbWords<16>& w, unsigned long long* x) {
  float v[RowShape<T>::V];
  sb_unpack_words<T, RowShape<T>::V>(w, v);
#pragma unroll
  for (int i = 0; i < RowShape<T>::V / 2; ++i) x[i] = pack_f32x2(v[2 * i], v[2 * i + 1]);
}

// The sums of a thread's share of a row of legal logits, in powers of two: with c = s / ln 2 and the reference R = c top, rounded,
//   sum = sum 2^(c x - R)   dist = sum 2^(c x - R) (c x - R),
// one fused multiply-add, one exponential and two additions per logit, two at a time.  The rounding of R is made good at the end.  Four batches
// of packs are on their way; a batch raises the reference first.  top_a and top_b: the largest of the even and of the odd packs.
template <typename T>
struct FastSums {
  float c, top_a, top_b, ref;
  unsigned long long sum, dist;
};
template <typename T>
__device__ __forceinline__ void lp_fast_raise(FastSums<T>& f) {
  const float ref = fmaxf(f.top_a, f.top_b) * f.c, d = f.ref - ref, e = exp2_approx(d);
  const unsigned long long d2 = pack_f32x2(d, d), e2 = pack_f32x2(e, e);
  fma_f32x2(f.dist, f.sum, d2);
  f.dist = mul_f32x2(f.dist, e2);
  f.sum = mul_f32x2(f.sum, e2);
  f.ref = ref;
}
template <typename T>
__device__ __forceinline__ void lp_fast_pack(FastSums<T>& f, const SbWords<16>& w) {
  unsigned long long x[RowShape<T>::V / 2];
  lp_pairs<T>(w, x);
  const unsigned long long c2 = pack_f32x2(f.c, f.c), ref2 = pack_f32x2(-f.ref, -f.ref);
#pragma unroll
  for (int i = 0; i < RowShape<T>::V / 2; ++i) {
    unsigned long long a2 = ref2;
    fma_f32x2(a2, x[i], c2);
    float a0, a1;
    unpack_f32x2(a2, a0, a1);
    const unsigned long long e2 = pack_f32x2(exp2_approx(a0), exp2_approx(a1));
    f.sum = add_f32x2(f.sum, e2);
    fma_f32x2(f.dist, e2, a2);
  }
}
template <typename T>
__device__ __forceinline__ ShareSums lp_fast_sums(const T* x, const RowShape<T>& shape, int first, int stride, float c) {
  constexpr int UNROLL = 4;
  const float low = lp_low<T>();
  FastSums<T> f = {c, low, low, low * c, 0ull, 0ull};
  if (first < shape.head + shape.tail) {
    const float v = max_nan(sb_to_f32<T>(x[shape.single(first)]), low);
    f.top_a = fmaxf(low, v);
    f.ref = f.top_a * c;
    const float a = fmaf(v, c, -f.ref), e = exp2_approx(a);
    f.sum = pack_f32x2(e, 0.f);
    f.dist = pack_f32x2(e * a, 0.f);
  }
  const T* from = x + shape.head;
  // Packs that are not there hold -inf.
  auto load = [&](SbWords<16>* w, int p) {
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      w[u].v.x = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
      w[u].v.y = w[u].v.z = w[u].v.w = w[u].v.x;
      sb_load_words(w[u], from + (long long)(p + u * stride) * RowShape<T>::V, p + u * stride < shape.packs);
    }
  };
  auto take = [&](SbWords<16>* w) {
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      lp_lift<T>(w[u]);
      if (u % 2 == 0) f.top_a = fmaxf(f.top_a, lp_largest<T>(w[u]));
      else f.top_b = fmaxf(f.top_b, lp_largest<T>(w[u]));
    }
    lp_fast_raise(f);
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) lp_fast_pack(f, w[u]);
  };
  SbWords<16> now[UNROLL], next[UNROLL];
  load(now, first);
  for (int p = first; p < shape.packs; p += UNROLL * stride) {
    load(next, p + UNROLL * stride);
    take(now);
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) now[u] = next[u];
  }
  float s0, s1, d0, d1;
  unpack_f32x2(f.sum, s0, s1);
  unpack_f32x2(f.dist, d0, d1);
  RowSums r;
  r.top = fmaxf(f.top_a, f.top_b);
  // c top is ref + rest.  (Far from zero the rest is large: such a share counts only in rows that take the exact sums, or not at all.)
  const float rest = fminf(fmaxf(fmaf(r.top, c, -f.ref), -60.f), 60.f), back = exp2_approx(-rest);
  r.sum = (s0 + s1) * back;
  r.dist = (d0 + d1 - rest * (s0 + s1)) * back;
  return {r, f.top_a, f.top_b};
}
// The fast sums of a row are right where its largest logit is neither so low (first) that what was lifted has weight beside it nor so far
// up (second) that the reference's rounding, 2^-4 of a power of two, is not made good to the last bits.
constexpr float LP_FAST_MOST = 1048576.f;
template <typename T>
__device__ __forceinline__ bool lp_not_low(float top, float c) { return (top - lp_low<T>()) * c >= 60.f && top * c >= -LP_FAST_MOST; }
__device__ __forceinline__ bool lp_too_high(float top, float c) { return top * c > LP_FAST_MOST || c > LP_FAST_MOST; }

// -inf where the bytes of a mask forbid a pack's columns.
template <typename T>
__device__ __forceinline__ void lp_mask_pack(float* x, const uint8_t* mask) {
  constexpr int V = RowShape<T>::V;
  uint8_t m[V];
  if (reinterpret_cast<uintptr_t>(mask) % V == 0) {
    SbWords<V> w;
    sb_load_words(w, mask, true);
    memcpy(m, &w, V);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) m[i] = mask[i];
  }
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (m[i] == 0) x[i] = -INFINITY;
}

// The same sums one logit at a time, under a mask or where the fast ones do not hold.
template <typename T>
__device__ __noinline__ ShareSums lp_exact_sums(const T* x, const uint8_t* mask, int cols, int first, int stride, float c) {
  const RowShape<T> shape(x, cols);
  constexpr int V = RowShape<T>::V;
  RowSums r = {LP_LOWEST, 0.f, 0.f};
  float top_a = LP_LOWEST, top_b = LP_LOWEST;
  if (first < shape.head + shape.tail) {
    const float v = lp_logit<T>(x, mask, shape.single(first));
    r.top = top_a = fmaxf(r.top, v);
    lp_take<1>(r, &v, c);
  }
  constexpr int UNROLL = 4;
  const bool whole = mask && reinterpret_cast<uintptr_t>(mask + shape.head) % V == 0;
  for (int p0 = first; p0 < shape.packs; p0 += UNROLL * stride) {
    SbWords<16> w[UNROLL];
    SbWords<V> m[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int p = p0 + u * stride;
      w[u].v = make_uint4(0u, 0u, 0u, 0u);
      sb_load_words(w[u], x + shape.column(p < shape.packs ? p : p0), true);
      memset(&m[u], 1, V);
      sb_load_words(m[u], mask + shape.column(p < shape.packs ? p : p0), whole);
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int p = p0 + u * stride;
      if (p >= shape.packs) break;
      float v[V];
      sb_unpack_words<T, V>(w[u], v);
      if (mask && !whole) {
        lp_mask_pack<T>(v, mask + shape.column(p));
      } else {
        uint8_t legal[V];
        memcpy(legal, &m[u], V);
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (legal[i] == 0) v[i] = -INFINITY;
      }
      float most = LP_LOWEST;
#pragma unroll
      for (int i = 0; i < V; ++i) most = fmaxf(most, v[i]);
      if (u % 2 == 0) top_a = fmaxf(top_a, most);
      else top_b = fmaxf(top_b, most);
      lp_raise(r, fmaxf(r.top, most), c);
      lp_take<V>(r, v, c);
    }
  }
  return {r, top_a, top_b};
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
__device__ __forceinline__ void lp_rank(unsigned long long* candidates, int n, unsigned long long* best, int top, int first, int threads) {
  for (int i = first; i < n; i += threads) {
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
// 4096 x 50001 in bf16 with 8 alternatives: 97 to 107 us where the bytes take 62.5; without alternatives 80 to 82, bound by the exponentials' unit (60 % busy)
// and the issue (57 %) as much as by memory.
template <typename T, int NT, bool MASKED, bool CLUSTER>
__global__ void __launch_bounds__(NT, NT == 512 ? 2 : 1280 / NT) log_probs_long_kernel(LogProbArgs g) {
  constexpr int V = RowShape<T>::V, WARPS = NT / 32;
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
  const float c = lp_factor(g.scale);
  for (long long row = blockIdx.y; row < g.rows; row += gridDim.y) {
    const T* x = reinterpret_cast<const T*>(g.logits) + row * g.ld;
    const uint8_t* mask = MASKED ? g.mask + row * g.mask_cols : nullptr;
    const RowShape<T> shape(x, g.cols);
    const int stride = NT * blocks, first = rank * NT + tid;
    const int singles = shape.head + shape.tail;               // fewer than 2 V: the first threads of the first block have one each
    long long token = -1;
    float token_logit = 0.f;
    if (g.out && first == 0) {
      token = lp_token(g.tokens, g.wide_tokens, row);
      if (token >= 0 && token < g.cols) token_logit = lp_logit<T>(x, mask, (int)token);
    }
    ShareSums mine = MASKED ? lp_exact_sums<T>(x, mask, g.cols, first, stride, c) : lp_fast_sums<T>(x, shape, first, stride, c);
    if (!MASKED) {
      // The same decision in all blocks of a row: one whose own share has no logit to speak of lets the others have theirs.
      const bool low = !__syncthreads_or(lp_not_low<T>(mine.r.top, c));
      if (__syncthreads_or(lp_too_high(mine.r.top, c)) || low) mine = lp_exact_sums<T>(x, nullptr, g.cols, first, stride, c);
    }
    RowSums r = mine.r;
    const float own = r.top;
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
    if (g.top > 0) largest[tid] = own;
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
            if (reach <= g.top + 8) break;
          }
        }
        // The key as a number; where fewer threads than alternatives have a logit to speak of everything counts.
        const float b = __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
        if (lane == 0) bound = key <= lp_key(lp_low<T>()) ? LP_LOWEST : b;
      }
      __syncthreads();
      const float least = bound;
      if (own >= least) hot[atomicAdd(&hot_count, 1)] = tid;
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
        lp_rank(candidates, n, best, g.top, tid, NT);
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
      // What was read of the others has arrived before they go on, and what this block's warps counted is seen by all of them.
      cluster_sync_all();
      if (rank == 0 && g.top > 0) {
        const int n = candidate_count;
        if (tid < LP_MAX_TOP) best[tid] = 0ull;
        __syncthreads();
        lp_rank(candidates, n, best, g.top, tid, NT);
        __syncthreads();
      }
    }
    if (rank == 0) {
      const float log_sum = all.sum == 0.f ? INFINITY : logf(all.sum);
      if (tid == 0) lp_finish(g, row, all, log_sum, token_logit, token);
      if (tid < g.top) lp_alternative(g, row, tid, lp_place_logit(best[tid]), best[tid] == 0ull ? -1 : lp_place_column(best[tid]), all.top, log_sum);
    }
  }
}

// Rows of middle length, and long ones where there are many: a warp per row, which needs no barrier.  The same steps; a lane's even and odd
// packs have a largest logit each, so that there are 64 to bound the alternatives by.
constexpr int LP_WARP_CANDIDATES = 160;
template <typename T, bool MASKED>
__global__ void __launch_bounds__(128, 8) log_probs_warp_kernel(LogProbArgs g) {
  constexpr int V = RowShape<T>::V;
  __shared__ __align__(16) unsigned long long all_candidates[4][LP_WARP_CANDIDATES];
  __shared__ unsigned long long all_best[4][LP_MAX_TOP];
  __shared__ uint8_t all_hot[4][64];
  __shared__ int counts[4];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  unsigned long long* candidates = all_candidates[warp];
  unsigned long long* best = all_best[warp];
  uint8_t* hot = all_hot[warp];
  sb_grid_dependency_wait();
  sb_grid_dependents_launch();
  const float c = lp_factor(g.scale);
  for (long long row = (long long)blockIdx.x * 4 + warp; row < g.rows; row += (long long)gridDim.x * 4) {
    const T* x = reinterpret_cast<const T*>(g.logits) + row * g.ld;
    const uint8_t* mask = MASKED ? g.mask + row * g.mask_cols : nullptr;
    const RowShape<T> shape(x, g.cols);
    const int singles = shape.head + shape.tail;
    long long token = -1;
    float token_logit = 0.f;
    if (g.out && lane == 0) {
      token = lp_token(g.tokens, g.wide_tokens, row);
      if (token >= 0 && token < g.cols) token_logit = lp_logit<T>(x, mask, (int)token);
    }
    ShareSums mine = MASKED ? lp_exact_sums<T>(x, mask, g.cols, lane, 32, c) : lp_fast_sums<T>(x, shape, lane, 32, c);
    if (!MASKED) {
      const bool low = !__any_sync(0xffffffffu, lp_not_low<T>(mine.r.top, c));
      if (__any_sync(0xffffffffu, lp_too_high(mine.r.top, c)) || low) mine = lp_exact_sums<T>(x, nullptr, g.cols, lane, 32, c);
    }
    RowSums r = mine.r;
    const float top_a = mine.top_a, top_b = mine.top_b;
    float top = r.top;
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    lp_raise(r, top, c);
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      r.sum += __shfl_xor_sync(0xffffffffu, r.sum, o);
      r.dist += __shfl_xor_sync(0xffffffffu, r.dist, o);
    }
    const float log_sum = r.sum == 0.f ? INFINITY : logf(r.sum);
    if (lane == 0) lp_finish(g, row, r, log_sum, token_logit, token);
    if (g.top == 0) continue;
    const uint32_t key_a = lp_key(top_a), key_b = lp_key(top_b);
    const uint32_t low = __reduce_min_sync(0xffffffffu, min(key_a, key_b)), high = __reduce_max_sync(0xffffffffu, max(key_a, key_b));
    const int alike = __clz((int)(low ^ high));
    uint32_t key = alike == 32 ? low : low & ~(0xffffffffu >> alike);
    for (int bit = 31 - alike; bit >= 0; --bit) {
      const uint32_t tried = key | 1u << bit;
      const int reach = __popc(__ballot_sync(0xffffffffu, key_a >= tried)) + __popc(__ballot_sync(0xffffffffu, key_b >= tried));
      if (reach >= g.top) {
        key = tried;
        if (reach <= g.top + 2) break;
      }
    }
    const float least = key <= lp_key(lp_low<T>()) ? LP_LOWEST : __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
    const uint32_t hot_a = __ballot_sync(0xffffffffu, top_a >= least), hot_b = __ballot_sync(0xffffffffu, top_b >= least);
    __syncwarp();                                // what the row before left has been read
    if (hot_a >> lane & 1u) hot[__popc(hot_a & ((1u << lane) - 1u))] = (uint8_t)lane;
    if (hot_b >> lane & 1u) hot[__popc(hot_a) + __popc(hot_b & ((1u << lane) - 1u))] = (uint8_t)(32 + lane);
    if (lane == 0) counts[warp] = 0;
    for (int i = lane; i < g.top; i += 32) best[i] = 0ull;
    __syncwarp();
    auto candidate = [&](float v, int j) {
      if (v >= least && v > -INFINITY) {
        const int at = atomicAdd(&counts[warp], 1);
        if (at < LP_WARP_CANDIDATES) candidates[at] = lp_place(v, j);
      }
    };
    // A share: every second pack of a lane's; the single element goes with the even ones.
    const int each = ((shape.packs + 31) / 32 + 1) / 2 + 1, items = (__popc(hot_a) + __popc(hot_b)) * each;
    for (int item = lane; item < items; item += 32) {
      const int who = hot[item / each], k = item % each, pack = 32 * (2 * k + (who >> 5)) + (who & 31);
      if (k == each - 1) {
        if (who < singles) candidate(lp_logit<T>(x, mask, shape.single(who)), shape.single(who));
      } else if (pack < shape.packs) {
        SbWords<16> w;
        sb_load_kept(w, x + shape.column(pack), true);
        if (MASKED || lp_largest<T>(w) >= least) {
          float v[V];
          sb_unpack_words<T, V>(w, v);
          if (MASKED) lp_mask_pack<T>(v, mask + shape.column(pack));
#pragma unroll
          for (int i = 0; i < V; ++i) candidate(v[i], shape.column(pack) + i);
        }
      }
    }
    __syncwarp();
    const int n = counts[warp];
    if (n <= LP_WARP_CANDIDATES) {
      lp_rank(candidates, n, best, g.top, lane, 32);
    } else {
      unsigned long long last = ~0ull;
      for (int i = 0; i < g.top; ++i) {
        unsigned long long next = 0ull;
        auto look = [&](float v, int j) {
          const unsigned long long place = lp_place(v, j);
          if (v > -INFINITY && place < last && place > next) next = place;
        };
        if (lane < singles) look(lp_logit<T>(x, mask, shape.single(lane)), shape.single(lane));
        for (int p = lane; p < shape.packs; p += 32) {
          SbWords<16> w;
          sb_load_kept(w, x + shape.column(p), true);
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
        if (lane == 0) best[i] = next;
        last = next;
      }
    }
    __syncwarp();
    for (int i = lane; i < g.top; i += 32) lp_alternative(g, row, i, lp_place_logit(best[i]), best[i] == 0ull ? -1 : lp_place_column(best[i]), top, log_sum);
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

// Bound by memory: 4096 x 50001 in bf16 140 us, 5.8 TB/s read and written.
// Long rows, NT threads each: packs of 16 bytes, several on their way; the blocks of a column of the grid share the rows.  With c = s / ln 2 and
// log p_j / ln 2 = c x_j - (ref + rest), where ref is rounded, a logit takes a fused multiply-add, an exponential, another multiply-add and a product, two at a
// time: the constants have the rest and all factors in them.
template <typename T, bool MASKED, int NT>
__global__ void __launch_bounds__(256) log_probs_grad_long_kernel(LogProbGradArgs g) {
  constexpr int V = RowShape<T>::V, UNROLL = 4;
  sb_grid_dependency_wait();
  sb_grid_dependents_launch();
  const int first = NT == 256 ? blockIdx.x * 256 + threadIdx.x : threadIdx.x % NT, stride = NT == 256 ? gridDim.x * 256 : NT;
  const float c = lp_factor(g.scale);
  for (long long row = NT == 256 ? blockIdx.y : (long long)blockIdx.x * (256 / NT) + threadIdx.x / NT; row < g.rows;
       row += NT == 256 ? gridDim.y : (long long)gridDim.x * (256 / NT)) {
    const RowGrad r = lp_row_grad(g, row);
    const T* x = reinterpret_cast<const T*>(g.logits) + row * g.ld;
    const uint8_t* mask = MASKED ? g.mask + row * g.mask_cols : nullptr;
    T* d = reinterpret_cast<T*>(g.dlogits) + row * g.ldd;
    const RowShape<T> shape(x, g.cols);
    const bool alike = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(d)) & 15u) == 0;
    if (first < shape.head + shape.tail) lp_grad_one<T>(r, x, mask, d, shape.single(first), g.cols);
    // (Up to 2^31 - 1 columns: a step behind the last one is beyond 32 bits.)
    for (long long j = (long long)g.cols + first; j < g.mask_cols; j += stride) d[j] = sb_from_f32<T>(0.f);
    const float ref = fmaf(r.top, c, r.log_sum * LP_LOG2E), rest = fmaf(r.top, c, -ref) + r.log_sum * LP_LOG2E, back = -r.scale * exp2_approx(-rest);
    const float h = back * r.h * (1.f / LP_LOG2E), k = back * fmaf(r.h, -rest * (1.f / LP_LOG2E), r.c);
    // The short way holds where the lifted logits come out as 0 and no product leaves fp32's range: not that of a lifted logit's logarithm, which
    // is the largest, and h either, as it would be infinite beside a probability of 0.
    const bool fast = fabsf(r.top) * c <= LP_FAST_MOST && c <= LP_FAST_MOST && (r.top - lp_low<T>()) * c >= 200.f && r.log_sum <= LP_FAST_MOST &&
                      -lp_low<T>() * c * fabsf(h) < 1e37f && fabsf(r.c) < 1e30f;
    const unsigned long long c2 = pack_f32x2(c, c), ref2 = pack_f32x2(-ref, -ref), h2 = pack_f32x2(h, h), k2 = pack_f32x2(k, k);
    for (int p0 = first; p0 < shape.packs; p0 += UNROLL * stride) {
      SbWords<16> w[UNROLL];
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) lp_load_once(w[u], x + shape.column(p0 + u * stride < shape.packs ? p0 + u * stride : p0), true);
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) {
        if (p0 + u * stride >= shape.packs) break;
        const int j = shape.column(p0 + u * stride);
        float v[V];
        if (fast) {
          unsigned long long pairs[V / 2];
          lp_lift<T>(w[u]);
          lp_pairs<T>(w[u], pairs);
#pragma unroll
          for (int i = 0; i < V / 2; ++i) {
            unsigned long long a2 = ref2, q2 = k2;
            fma_f32x2(a2, pairs[i], c2);
            fma_f32x2(q2, a2, h2);
            float a0, a1;
            unpack_f32x2(a2, a0, a1);
            unpack_f32x2(mul_f32x2(pack_f32x2(exp2_approx(a0), exp2_approx(a1)), q2), v[2 * i], v[2 * i + 1]);
          }
        } else {
          sb_unpack_words<T, V>(w[u], v);
#pragma unroll
          for (int i = 0; i < V; ++i) v[i] = lp_grad(r, v[i]);
        }
        if ((unsigned)(r.token - j) < (unsigned)V) {
#pragma unroll
          for (int i = 0; i < V; ++i)
            if (j + i == r.token) v[i] += r.a;
        }
        if (MASKED) {
          float legal[V] = {};
          lp_mask_pack<T>(legal, mask + j);
#pragma unroll
          for (int i = 0; i < V; ++i) v[i] = legal[i] == 0.f ? v[i] : 0.f;
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

int lp_args_ok(const char* who, const void* logits, long long ld, int dtype, long long rows, int cols, int prefix, float scale, const void* tokens,
               int index_dtype) {
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

// What takes a row: `threads` of a warp with `columns` each in registers (0: in one pass over memory), or a block of them, and `blocks` that share a row.
struct LogProbForm {
  int threads, columns, blocks;
};
LogProbForm log_probs_form(long long rows, int cols, int top) {
  // Few lanes with many columns each: their rounds cost by the lane.  us, 65536 rows: 10 columns (fp32, 2 alternatives) with 4 / 2 lanes 7.5 / 5.5; 20 with
  // 8 / 4 14.7 / 8.1; 64 (bf16, 2) with 8 / 4 / 2 15.0 / 12.3 / 13.5; 100000 rows: 128 (bf16, none) with 32 / 8 / 4 46.8 / 20.8 / 14.9, with 32
  // alternatives by warps, as below / 8 / 4 413 / 212 / 172; 200 (2) with 32 / 16 / 8 84.5 / 66.6 / 46.7.
  if (cols <= 16) return {2, 8, 1};
  if (cols <= 32) return {4, 8, 1};
  if (cols <= 64) return {4, 16, 1};
  if (cols <= 128) return {4, 32, 1};
  // Rounds cost by the alternative, the warps' bound costs once: 250 columns with 16 alternatives 237 (16 lanes) / 168; 500 columns with none, 2 or 7 of
  // them 28 / 41, 53 / 88, 59 / 41 (32768 rows of fp32); 1000 with 2 of them 54 / 45.
  if (cols <= 256 && top <= 7) return {8, 32, 1};
  if (cols <= 512 && top <= 3) return {16, 32, 1};
  // Warps or blocks, 8 alternatives: 32768 x 2048 69 / 152, 16384 x 8192 94 / 98, 8192 x 16384 93 / 80, 600 x 4096 11.7 / 9.3.
  if (cols <= 1024 || (cols <= 8192 && rows >= 16LL * sb_sm_count())) return {32, 0, 1};
  // A cluster per row where rows are few, all of them resident at once: 35 x 41654 with 3 alternatives in clusters of 8, which the chip's parts hold 32
  // of, 16.3, of 4 9.5; 70 rows 12.1 (4), 9.1 (2).
  int blocks = 1;
  while (blocks < 8 && rows * blocks * 2 <= 3LL * sb_sm_count() / 2 && cols / (2 * blocks) >= 4096) blocks *= 2;
  if (blocks > 1) return {512, 0, blocks};
  // Threads of a row, 8 alternatives, 128 / 256 / 512: 4096 x 20000 53 / 61 / 114, 4096 x 50001 114 / 103 / 139, 1024 x 130000 80 / 73 / 66.
  return {cols <= 24576 ? 128 : cols <= 98304 ? 256 : 512, 0, 1};
}

template <typename T>
int launch_log_probs(const LogProbArgs& g, cudaStream_t s) {
  const LogProbForm form = log_probs_form(g.rows, g.cols, g.top);
  if (form.columns > 0) {
    if (form.threads == 2) return launch_log_probs_short<T, 2, 8>(g, s);
    if (form.threads == 4)
      return form.columns == 8 ? launch_log_probs_short<T, 4, 8>(g, s) : form.columns == 16 ? launch_log_probs_short<T, 4, 16>(g, s) : launch_log_probs_short<T, 4, 32>(g, s);
    return form.threads == 8 ? launch_log_probs_short<T, 8, 32>(g, s) : launch_log_probs_short<T, 16, 32>(g, s);
  }
  if (form.threads == 32) {
    const long long blocks = (g.rows + 3) / 4, most = 64LL * sb_sm_count();
    const dim3 grid((unsigned)(blocks < most ? blocks : most));
    if (g.mask) SB_CUDA(sb_launch(log_probs_warp_kernel<T, true>, grid, dim3(128), 0, s, 1, g));
    else SB_CUDA(sb_launch(log_probs_warp_kernel<T, false>, grid, dim3(128), 0, s, 1, g));
    SB_COUNT_LAUNCH();
    return SB_OK;
  }
  if (form.blocks > 1) return launch_log_probs_long<T, 512, true>(g, form.blocks, s);
  if (form.threads == 128) return launch_log_probs_long<T, 128, false>(g, 1, s);
  if (form.threads == 256) return launch_log_probs_long<T, 256, false>(g, 1, s);
  return launch_log_probs_long<T, 512, false>(g, 1, s);
}

template <typename T>
int launch_log_probs_grad(const LogProbGradArgs& g, cudaStream_t s) {
  if (g.mask_cols <= 64) {
    const int lanes = g.mask_cols <= 16 ? 4 : 8;
    const long long blocks = (g.rows * lanes + 255) / 256, most = 32LL * sb_sm_count();
    const dim3 grid((unsigned)(blocks < most ? blocks : most));
    if (lanes == 4) SB_CUDA(sb_launch(log_probs_grad_short_kernel<T, 4>, grid, dim3(256), 0, s, 1, g));
    else SB_CUDA(sb_launch(log_probs_grad_short_kernel<T, 8>, grid, dim3(256), 0, s, 1, g));
    SB_COUNT_LAUNCH();
    return SB_OK;
  }
  // A warp per row where that keeps the chip busy.
  if (g.mask_cols <= 4096 && g.rows * 8 >= (long long)sb_sm_count() * (g.mask_cols / 64)) {
    const long long blocks = (g.rows + 7) / 8, most = 64LL * sb_sm_count();
    const dim3 grid((unsigned)(blocks < most ? blocks : most));
    if (g.mask) SB_CUDA(sb_launch(log_probs_grad_long_kernel<T, true, 32>, grid, dim3(256), 0, s, 1, g));
    else SB_CUDA(sb_launch(log_probs_grad_long_kernel<T, false, 32>, grid, dim3(256), 0, s, 1, g));
    SB_COUNT_LAUNCH();
    return SB_OK;
  }
  // Enough blocks for the chip where rows are few, each with a batch of packs per thread at least.
  const int batch = 256 * 4 * (16 / (int)sizeof(T));
  long long across = (8LL * sb_sm_count() + g.rows - 1) / g.rows;
  const long long most_across = ((long long)g.mask_cols + batch - 1) / batch;
  if (across > most_across) across = most_across;
  const dim3 grid((unsigned)across, (unsigned)(g.rows < 65535 ? g.rows : 65535));
  if (g.mask) SB_CUDA(sb_launch(log_probs_grad_long_kernel<T, true, 256>, grid, dim3(256), 0, s, 1, g));
  else SB_CUDA(sb_launch(log_probs_grad_long_kernel<T, false, 256>, grid, dim3(256), 0, s, 1, g));
  SB_COUNT_LAUNCH();
  return SB_OK;
}

}  // namespace

extern "C" {

int sb_log_probs(const void* logits, long long ld, int dtype, long long rows, int cols, const uint8_t* mask, int prefix, float scale,
                 const void* tokens, int index_dtype, float* out, float* entropy, float* stats, int top, float* top_values,
                 int32_t* top_tokens, void* stream) {
  const char* who = "sb_log_probs";
  int rc = lp_args_ok(who, logits, ld, dtype, rows, cols, prefix, scale, tokens, index_dtype);
  if (rc != SB_OK) return rc;
  if (top < 0) return sb_fail(SB_ERR_BAD_ARG, "%s: negative size", who);
  if (top > LP_MAX_TOP) return sb_fail(SB_ERR_TOO_LARGE, "%s: at most %d alternatives (got %d)", who, LP_MAX_TOP, top);
  if (rows == 0) return SB_OK;
  if (out && !tokens) return sb_fail(SB_ERR_BAD_ARG, "%s: log probabilities of no tokens", who);
  if (top > 0 && !top_values && !top_tokens) return sb_fail(SB_ERR_BAD_ARG, "%s: nowhere to put %d alternatives", who, top);
  if (!lp_words(out) || !lp_words(entropy) || !lp_words(stats) || !lp_words(top_values) || !lp_words(top_tokens))
    return sb_fail(SB_ERR_MISALIGNED, "%s: a pointer is not aligned to its element size", who);
  for (const void* o : {(const void*)out, (const void*)entropy, (const void*)stats, (const void*)top_values, (const void*)top_tokens})
    if (o && cols > 0 && (o == logits || o == (const void*)mask)) return sb_fail(SB_ERR_BAD_ARG, "%s: an output in the place of the logits or the mask", who);
  LogProbArgs g;
  memset(&g, 0, sizeof(g));
  g.logits = logits; g.ld = ld; g.rows = rows; g.cols = prefix >= 0 ? prefix : cols; g.mask_cols = cols;
  g.mask = prefix >= 0 ? nullptr : mask; g.scale = scale; g.tokens = tokens; g.wide_tokens = index_dtype == SB_I64; g.out = out; g.entropy = entropy; g.stats = stats;
  g.top = top; g.top_values = top_values; g.top_tokens = top_tokens;
  cudaStream_t s = (cudaStream_t)stream;
  return dtype == SB_F32 ? launch_log_probs<float>(g, s)
         : dtype == SB_BF16 ? launch_log_probs<__nv_bfloat16>(g, s) : launch_log_probs<__half>(g, s);
}

int sb_log_probs_plan(long long rows, int cols, int top, int* plan) {
  const char* who = "sb_log_probs_plan";
  if (!plan) return sb_fail(SB_ERR_BAD_ARG, "%s: null output", who);
  if (rows <= 0 || cols <= 0 || top < 0 || top > LP_MAX_TOP) return sb_fail(SB_ERR_BAD_ARG, "%s: sizes of nothing, or more than %d alternatives", who, LP_MAX_TOP);
  const LogProbForm form = log_probs_form(rows, cols, top);
  plan[0] = form.threads;
  plan[1] = form.columns;
  plan[2] = form.blocks;
  return SB_OK;
}

int sb_log_probs_grad(const void* logits, long long ld, int dtype, long long rows, int cols, const uint8_t* mask, int prefix, float scale,
                      const void* tokens, int index_dtype, const float* stats, const float* dout, const float* entropy,
                      const float* dentropy, void* dlogits, long long ldd, void* stream) {
  const char* who = "sb_log_probs_grad";
  int rc = lp_args_ok(who, logits, ld, dtype, rows, cols, prefix, scale, tokens, index_dtype);
  if (rc != SB_OK) return rc;
  if (rows == 0 || cols == 0) return SB_OK;
  if (!dlogits || !stats) return sb_fail(SB_ERR_BAD_ARG, "%s: null pointer", who);
  if (dout && !tokens) return sb_fail(SB_ERR_BAD_ARG, "%s: a gradient of the log probabilities of no tokens", who);
  if (dentropy && !entropy) return sb_fail(SB_ERR_BAD_ARG, "%s: a gradient of the entropy needs the entropy", who);
  if (ldd < cols) return sb_fail(SB_ERR_BAD_ARG, "%s: a row pitch of %lld is shorter than the %d columns", who, ldd, cols);
  if (reinterpret_cast<uintptr_t>(dlogits) % (size_t)sb_dtype_size(dtype) != 0 || !lp_words(stats) || !lp_words(dout) || !lp_words(entropy) ||
      !lp_words(dentropy))
    return sb_fail(SB_ERR_MISALIGNED, "%s: a pointer is not aligned to its element size", who);
  if (dlogits == logits && rows > 1 && ldd != ld) return sb_fail(SB_ERR_BAD_ARG, "%s: gradients in the place of the logits have their row pitch", who);
  for (const void* i : {(const void*)mask, tokens, (const void*)stats, (const void*)dout, (const void*)entropy, (const void*)dentropy})
    if (i == dlogits) return sb_fail(SB_ERR_BAD_ARG, "%s: gradients in the place of another input than the logits", who);
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
