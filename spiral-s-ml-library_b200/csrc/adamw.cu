// One AdamW step over many tensors, states in 32 bits or in 8.
//
//   g = grad_scale * grad;  m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g g
//   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// All tensors of a call go through one launch (up to 400; more take further launches): their descriptors travel as a
// kernel parameter, so that nothing is kept on the device between calls, and a block finds its tensor by its number.
//
// States in 8 bits are E4M3 codes with one fp32 scale per 256 elements (the largest magnitude of the block / 448).  Held
// are m and r = sqrt(v): r has half the range of exponents that v has.  Rounding an average that moves by a thousandth
// per step to the nearest of codes that lie up to an eighth apart would leave it where it is, so a magnitude is rounded up
// with the probability of the part that is cut off: 20 bits of noise, a hash of the element's index and the caller's seed,
// are added below the code's last bit.  No positive r becomes zero, since the next step divides by it.
//
// The arithmetic of both forms is written out operation by operation (no contraction to fused multiply-adds): a state
// that is rounded to 8 bits is then a function that anyone can recompute.
#include "common.cuh"
#include "vector_io.cuh"

#include <math.h>

#include <type_traits>

namespace {

constexpr int AW_BLOCK = 256;                                // elements of a state that share a scale
constexpr int AW_CHUNK = 4096;                               // elements per thread block
constexpr float AW_TOP = 448.f;                              // the largest E4M3 value
constexpr float AW_FLOOR = 7.888609052210118e-31f;           // 2^-100: a block's largest magnitude is at least this
constexpr uint32_t AW_K1 = 0x9E3779B1u, AW_K2 = 0x6A09E667u, AW_K3 = 0xBB67AE85u, AW_K4 = 0xA54FF53Bu, AW_SALT = 0x3C6EF373u;

struct AdamwTensor {
  float* p;
  const void* g;
  void* m;                       // fp32 m, or E4M3 codes of m
  void* v;                       // fp32 v, or E4M3 codes of sqrt(v)
  float* ms;                     // scales per 256 elements
  float* vs;
  void* copy;                    // compute copy of the parameters, or NULL
  long long n;
};

struct AdamwHyper {
  float b1, c1, b2, c2;          // c = 1 - b
  float eps, keep;               // keep = 1 - lr wd
  float step;                    // lr / (1 - b1^t)
  float unbias;                  // 1 / sqrt(1 - b2^t)
  float grad_scale;
  uint32_t seed;
  int copy_dtype;
};

template <int MOST>
struct AdamwTable {
  AdamwTensor t[MOST];
  int first[MOST + 1];           // the tensor's first block
  int vec[MOST];                 // 1: every pointer allows 16-byte accesses
  int n;
  AdamwHyper h;
};

__device__ __forceinline__ uint32_t aw_noise(uint32_t index, uint32_t salted_seed) {
  uint32_t u = index * AW_K1 + salted_seed;
  u = (u ^ (u >> 16)) * AW_K3;
  u = (u ^ (u >> 15)) * AW_K4;
  return u >> 12;
}

// |y| <= 448 (or NaN) and 20 bits of noise -> E4M3.  |y| 2^-120 has the code's bits from bit 20 on, subnormals included.
template <bool FINITE>
__device__ __forceinline__ uint32_t aw_encode(float y, uint32_t noise) {
  const uint32_t u = __float_as_uint(__fmul_rn(fabsf(y), 7.52316384526264e-37f));
  const uint32_t code = !FINITE && u > 0x7f800000u ? 127u : min((u + noise) >> 20, 126u);
  return code | (__float_as_uint(y) >> 31 << 7);
}
__device__ __forceinline__ bool aw_16bit(int dtype) { return dtype == SB_BF16 || dtype == SB_F16; }

__device__ __forceinline__ void aw_update(const AdamwHyper& h, float& p, float g, float& m, float& v, float& r) {
  g = __fmul_rn(g, h.grad_scale);
  m = __fadd_rn(__fmul_rn(m, h.b1), __fmul_rn(g, h.c1));
  v = __fadd_rn(__fmul_rn(v, h.b2), __fmul_rn(__fmul_rn(g, h.c2), g));
  r = __fsqrt_rn(v);
  const float d = __fdiv_rn(m, __fadd_rn(__fmul_rn(r, h.unbias), h.eps));
  p = __fsub_rn(__fmul_rn(p, h.keep), __fmul_rn(d, h.step));
}

// The same for two neighbours, two products per instruction; the sums stay scalar, because the assembler joins packed products
// and packed sums into multiply-adds, which round once instead of twice.
__device__ __forceinline__ void aw_scale2(float* x, const float* a, float b) {
  unpack_f32x2(mul_f32x2(pack_f32x2(a[0], a[1]), pack_f32x2(b, b)), x[0], x[1]);
}
__device__ __forceinline__ void aw_update2(const AdamwHyper& h, float* p, float* g, float* m, float* v, float* r) {
  float a[2], b[2], d[2];
  aw_scale2(g, g, h.grad_scale);
  aw_scale2(a, m, h.b1);
  aw_scale2(b, g, h.c1);
#pragma unroll
  for (int k = 0; k < 2; ++k) m[k] = __fadd_rn(a[k], b[k]);
  aw_scale2(a, v, h.b2);
  aw_scale2(b, g, h.c2);
  unpack_f32x2(mul_f32x2(pack_f32x2(b[0], b[1]), pack_f32x2(g[0], g[1])), b[0], b[1]);
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    v[k] = __fadd_rn(a[k], b[k]);
    r[k] = __fsqrt_rn(v[k]);
  }
  aw_scale2(a, r, h.unbias);
#pragma unroll
  for (int k = 0; k < 2; ++k) d[k] = __fdiv_rn(m[k], __fadd_rn(a[k], h.eps));
  aw_scale2(a, p, h.keep);
  aw_scale2(b, d, h.step);
#pragma unroll
  for (int k = 0; k < 2; ++k) p[k] = __fsub_rn(a[k], b[k]);
}

__device__ __forceinline__ float aw_round_tf32(float v) {
  uint32_t u = __float_as_uint(v);
  if ((u & 0x7f800000u) == 0x7f800000u) return v;
  return __uint_as_float((u + 0x0fffu + ((u >> 13) & 1u)) & 0xffffe000u);
}

template <int V>
__device__ __forceinline__ void aw_store_copy(void* copy, int dtype, long long i, const float* p) {
  if (dtype == SB_BF16) sb_store_f32<__nv_bfloat16, V>((__nv_bfloat16*)copy + i, p);
  else if (dtype == SB_F16) sb_store_f32<__half, V>((__half*)copy + i, p);
  else if constexpr (V <= 4) {
    float t[V];
#pragma unroll
    for (int k = 0; k < V; ++k) t[k] = dtype == SB_TF32 ? aw_round_tf32(p[k]) : p[k];
    sb_store_f32<float, V>((float*)copy + i, t);
  }
}

template <typename G, int V>
__device__ __forceinline__ void adamw_wide(const AdamwTensor& t, const AdamwHyper& h, long long begin, long long end) {
  for (long long i = begin + threadIdx.x * V; i < end; i += blockDim.x * V) {
    float p[V], g[V], m[V], v[V], r;
    sb_unpack<float, V>(sb_load_pack<float, V>(t.p + i), p);
    sb_unpack<G, V>(sb_load_pack<G, V>((const G*)t.g + i), g);
    sb_unpack<float, V>(sb_load_pack<float, V>((const float*)t.m + i), m);
    sb_unpack<float, V>(sb_load_pack<float, V>((const float*)t.v + i), v);
#pragma unroll
    for (int k = 0; k < V; ++k) aw_update(h, p[k], g[k], m[k], v[k], r);
    sb_store_f32<float, V>(t.p + i, p);
    sb_store_f32<float, V>((float*)t.m + i, m);
    sb_store_f32<float, V>((float*)t.v + i, v);
    if (t.copy) aw_store_copy<V>(t.copy, h.copy_dtype, i, p);
  }
}

// E4M3 codes -> values times a scale, exactly: through fp16, which holds them all.
__device__ __forceinline__ void aw_decode4(uint32_t codes, float scale, float* x) {
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)(codes >> (16 * k))));
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
    x[2 * k] = __fmul_rn(f.x, scale);
    x[2 * k + 1] = __fmul_rn(f.y, scale);
  }
}

// A warp per 256-element block of the states, 8 elements per lane.  WIDE: neighbours, all loads of the block on their way at
// once; else, for any alignment and the tensor's last block, element 32 k + lane.
template <typename G, bool WIDE>
__device__ __forceinline__ void adamw_coded(const AdamwTensor& t, const AdamwHyper& h, long long b, long long end) {
  const int lane = threadIdx.x & 31;
  uint8_t* mc = (uint8_t*)t.m;
  uint8_t* vc = (uint8_t*)t.v;
  const long long i0 = WIDE ? b + 8 * lane : b + lane;
  constexpr int STEP = WIDE ? 1 : 32;
  const float ms = t.ms[b / AW_BLOCK], vs = t.vs[b / AW_BLOCK];
  float p[8], g[8], m[8], r[8];
  if (WIDE) {
    constexpr int GV = sizeof(G) == 2 ? 8 : 4;
    const uint2 cm = *reinterpret_cast<const uint2*>(mc + i0), cr = *reinterpret_cast<const uint2*>(vc + i0);
#pragma unroll
    for (int k = 0; k < 8; k += 4) sb_unpack<float, 4>(sb_load_pack<float, 4>(t.p + i0 + k), p + k);
#pragma unroll
    for (int k = 0; k < 8; k += GV) sb_unpack<G, GV>(sb_load_pack<G, GV>((const G*)t.g + i0 + k), g + k);
    aw_decode4(cm.x, ms, m);
    aw_decode4(cm.y, ms, m + 4);
    aw_decode4(cr.x, vs, r);
    aw_decode4(cr.y, vs, r + 4);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const long long i = i0 + k * STEP;
      const bool in = i < end;
      p[k] = in ? t.p[i] : 0.f;
      g[k] = in ? sb_to_f32<G>(((const G*)t.g)[i]) : 0.f;
      float x[4];
      aw_decode4(in ? mc[i] : 0u, ms, x);
      m[k] = in ? x[0] : 0.f;
      aw_decode4(in ? vc[i] : 0u, vs, x);
      r[k] = in ? x[0] : 0.f;
    }
  }
  uint32_t mx = 0u, rx = 0u;
#pragma unroll
  for (int k = 0; k < 8; k += 2) {
    float v[2] = {__fmul_rn(r[k], r[k]), __fmul_rn(r[k + 1], r[k + 1])};
    aw_update2(h, p + k, g + k, m + k, v, r + k);
  }
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    mx = max(mx, __float_as_uint(m[k]) & 0x7fffffffu);       // as integers: a NaN is the largest and stays
    rx = max(rx, __float_as_uint(r[k]) & 0x7fffffffu);
  }
  mx = __reduce_max_sync(0xffffffffu, mx);
  rx = __reduce_max_sync(0xffffffffu, rx);
  const float mm = __uint_as_float(max(mx, __float_as_uint(AW_FLOOR))), rm = __uint_as_float(max(rx, __float_as_uint(AW_FLOOR)));
  const float mi = __fdiv_rn(AW_TOP, mm), ri = __fdiv_rn(AW_TOP, rm);
  if (lane == 0) {
    t.ms[b / AW_BLOCK] = __fdiv_rn(mm, AW_TOP);
    t.vs[b / AW_BLOCK] = __fdiv_rn(rm, AW_TOP);
  }
  uint32_t cm[8], cr[8];
  auto encode = [&](auto finite) {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t i = (uint32_t)(i0 + k * STEP);
      cm[k] = aw_encode<decltype(finite)::value>(__fmul_rn(m[k], mi), aw_noise(i, h.seed));
      cr[k] = aw_encode<decltype(finite)::value>(__fmul_rn(r[k], ri), aw_noise(i, h.seed + AW_SALT));
      if (cr[k] == 0u && r[k] > 0.f) cr[k] = 1u;
    }
  };
  if (mm < INFINITY && rm < INFINITY) encode(std::true_type());   // the same for the whole warp
  else encode(std::false_type());
  if (WIDE) {
#pragma unroll
    for (int k = 0; k < 8; k += 4) sb_store_f32<float, 4>(t.p + i0 + k, p + k);
    auto four = [](const uint32_t* c) { return c[0] | c[1] << 8 | c[2] << 16 | c[3] << 24; };
    *reinterpret_cast<uint2*>(mc + i0) = make_uint2(four(cm), four(cm + 4));
    *reinterpret_cast<uint2*>(vc + i0) = make_uint2(four(cr), four(cr + 4));
    if (t.copy) {
      if (aw_16bit(h.copy_dtype)) {
        aw_store_copy<8>(t.copy, h.copy_dtype, i0, p);
      } else {
        aw_store_copy<4>(t.copy, h.copy_dtype, i0, p);
        aw_store_copy<4>(t.copy, h.copy_dtype, i0 + 4, p + 4);
      }
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const long long i = i0 + k * STEP;
      if (i < end) {
        t.p[i] = p[k];
        mc[i] = (uint8_t)cm[k];
        vc[i] = (uint8_t)cr[k];
        if (t.copy) aw_store_copy<1>(t.copy, h.copy_dtype, i, p + k);
      }
    }
  }
}

// 32-bit states: bound by memory, 100 M parameters 448 us, 6.7 TB/s.  8-bit states: by issue (73 % of the slots), 96 instructions
// per element, a third of them the square root and the division, a quarter the noise: 40 M parameters with bf16 gradients 146 us,
// 3.9 TB/s (174 without packed products and the finite path; 165 with the 80 registers that leave 24 warps per SM instead of 32).  At its 64
// registers the 8-bit form spills 20 (fp32 gradients) to 36 bytes (bf16).
template <typename G, bool CODED, int MOST>
__global__ void __launch_bounds__(256, 4) adamw_kernel(const __grid_constant__ AdamwTable<MOST> a) {
  sb_grid_dependency_wait();
  sb_grid_dependents_launch();
  int lo = 0, hi = a.n - 1;                                  // the last tensor whose first block is not behind this one
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (a.first[mid] <= (int)blockIdx.x) lo = mid;
    else hi = mid - 1;
  }
  const AdamwTensor& t = a.t[lo];
  const long long begin = (long long)((int)blockIdx.x - a.first[lo]) * AW_CHUNK;
  const long long end = begin + AW_CHUNK < t.n ? begin + AW_CHUNK : t.n;
  if (CODED) {
    for (long long b = begin + (threadIdx.x >> 5) * AW_BLOCK; b < end; b += (blockDim.x >> 5) * AW_BLOCK) {
      if (a.vec[lo] && b + AW_BLOCK <= end) adamw_coded<G, true>(t, a.h, b, end);
      else adamw_coded<G, false>(t, a.h, b, end);
    }
  } else if (a.vec[lo]) {
    const long long whole = begin + (end - begin) / 4 * 4;
    adamw_wide<G, 4>(t, a.h, begin, whole);
    adamw_wide<G, 1>(t, a.h, whole, end);
  } else {
    adamw_wide<G, 1>(t, a.h, begin, end);
  }
}

bool aw_aligned(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

template <typename G, bool CODED, int MOST>
int launch_adamw(const sb_adamw_tensor* d, int n, const AdamwHyper& h, int grad_size, int copy_size, cudaStream_t s) {
  AdamwTable<MOST> a;
  for (int at = 0; at < n;) {
    a.n = 0;
    a.h = h;
    long long blocks = 0;
    for (; at < n && a.n < MOST; ++at) {
      if (d[at].n == 0) continue;
      const long long mine = (d[at].n + AW_CHUNK - 1) / AW_CHUNK;
      if (blocks + mine > 0x7fffffffLL) break;
      AdamwTensor& t = a.t[a.n];
      t.p = d[at].param; t.g = d[at].grad; t.m = d[at].exp_avg; t.v = d[at].exp_avg_sq;
      t.ms = d[at].exp_avg_scale; t.vs = d[at].exp_avg_sq_scale; t.copy = d[at].copy; t.n = d[at].n;
      const size_t state = CODED ? 8 : 16;
      a.vec[a.n] = aw_aligned(t.p, 16) && aw_aligned(t.g, CODED && grad_size == 2 ? 16 : 4 * grad_size) && aw_aligned(t.m, state) &&
                   aw_aligned(t.v, state) && aw_aligned(t.copy, copy_size == 2 ? (CODED ? 16 : 8) : 16);
      a.first[a.n++] = (int)blocks;
      blocks += mine;
    }
    if (a.n == 0) break;
    a.first[a.n] = (int)blocks;
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3(256);
    cfg.stream = s;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = sb_pdl_enabled() ? 1 : 0;
    void* args[] = {&a};                                     // as sb_launch, without copies of the table
    SB_CUDA(cudaLaunchKernelExC(&cfg, (const void*)adamw_kernel<G, CODED, MOST>, args));
    SB_COUNT_LAUNCH();
  }
  return SB_OK;
}

template <typename G, bool CODED>
int launch_adamw_sized(const sb_adamw_tensor* d, int n, const AdamwHyper& h, int grad_size, int copy_size, cudaStream_t s) {
  if (n <= 40) return launch_adamw<G, CODED, 40>(d, n, h, grad_size, copy_size, s);
  return launch_adamw<G, CODED, 400>(d, n, h, grad_size, copy_size, s);
}

}  // namespace

extern "C" int sb_adamw_step(int n_tensors, const sb_adamw_tensor* tensors, int state_dtype, int grad_dtype, int copy_dtype,
                             const sb_adamw_hyper* hyper, void* stream) {
  const char* who = "sb_adamw_step";
  if (n_tensors < 0) return sb_fail(SB_ERR_BAD_ARG, "%s: negative number of tensors", who);
  if (state_dtype != SB_F32 && state_dtype != SB_E4M3) return sb_fail(SB_ERR_UNSUPPORTED, "%s: states are f32 or e4m3", who);
  if (grad_dtype != SB_F32 && grad_dtype != SB_BF16 && grad_dtype != SB_F16)
    return sb_fail(SB_ERR_UNSUPPORTED, "%s: gradients are f32, bf16 or f16", who);
  if (copy_dtype != SB_F32 && copy_dtype != SB_TF32 && copy_dtype != SB_BF16 && copy_dtype != SB_F16)
    return sb_fail(SB_ERR_UNSUPPORTED, "%s: copies are f32, tf32, bf16 or f16", who);
  if (n_tensors == 0) return SB_OK;
  if (!tensors || !hyper) return sb_fail(SB_ERR_BAD_ARG, "%s: null pointer", who);
  if (hyper->step < 1) return sb_fail(SB_ERR_BAD_ARG, "%s: steps are counted from 1 (got %lld)", who, hyper->step);
  if (!(hyper->beta1 >= 0. && hyper->beta1 < 1. && hyper->beta2 >= 0. && hyper->beta2 < 1.) || !(hyper->eps >= 0.))
    return sb_fail(SB_ERR_BAD_ARG, "%s: betas lie in [0, 1) and eps is not negative", who);
  const int gs = sb_dtype_size(grad_dtype), cs = sb_dtype_size(copy_dtype);
  const bool coded = state_dtype == SB_E4M3;
  for (int i = 0; i < n_tensors; ++i) {
    const sb_adamw_tensor& t = tensors[i];
    if (t.n < 0) return sb_fail(SB_ERR_BAD_ARG, "%s: tensor %d has a negative size", who, i);
    if (t.n == 0) continue;
    if (!t.param || !t.grad || !t.exp_avg || !t.exp_avg_sq) return sb_fail(SB_ERR_BAD_ARG, "%s: tensor %d has a null pointer", who, i);
    if (coded && (!t.exp_avg_scale || !t.exp_avg_sq_scale))
      return sb_fail(SB_ERR_BAD_ARG, "%s: tensor %d has 8-bit states without scales", who, i);
    if (!aw_aligned(t.param, 4) || !aw_aligned(t.grad, gs) || !aw_aligned(t.copy, cs) || !aw_aligned(t.exp_avg_scale, 4) ||
        !aw_aligned(t.exp_avg_sq_scale, 4) || (!coded && (!aw_aligned(t.exp_avg, 4) || !aw_aligned(t.exp_avg_sq, 4))))
      return sb_fail(SB_ERR_MISALIGNED, "%s: tensor %d has a pointer that is not aligned to its element size", who, i);
  }
  AdamwHyper h;
  h.b1 = (float)hyper->beta1; h.c1 = (float)(1. - hyper->beta1);
  h.b2 = (float)hyper->beta2; h.c2 = (float)(1. - hyper->beta2);
  h.eps = (float)hyper->eps; h.keep = (float)(1. - hyper->lr * hyper->weight_decay);
  h.step = (float)(hyper->lr / (1. - pow(hyper->beta1, (double)hyper->step)));
  h.unbias = (float)(1. / sqrt(1. - pow(hyper->beta2, (double)hyper->step)));
  h.grad_scale = (float)hyper->grad_scale;
  h.seed = hyper->seed * AW_K2;
  h.copy_dtype = copy_dtype;
  cudaStream_t s = (cudaStream_t)stream;
#define SB_ADAMW_BY_STATE(G)                                                              \
  (coded ? launch_adamw_sized<G, true>(tensors, n_tensors, h, gs, cs, s)                  \
         : launch_adamw_sized<G, false>(tensors, n_tensors, h, gs, cs, s))
  if (grad_dtype == SB_F32) return SB_ADAMW_BY_STATE(float);
  if (grad_dtype == SB_BF16) return SB_ADAMW_BY_STATE(__nv_bfloat16);
  return SB_ADAMW_BY_STATE(__half);
#undef SB_ADAMW_BY_STATE
}
