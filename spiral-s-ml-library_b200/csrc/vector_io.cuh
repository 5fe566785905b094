// Loads and stores of V neighbouring elements of a storage type as fp32 values, one aligned access each
// (V * sizeof(T) is 2, 4, 8 or 16 bytes), for the kernels that stream matrices through registers.
#pragma once

#include "common.cuh"

template <typename T>
__device__ __forceinline__ float sb_to_f32(T v);
template <>
__device__ __forceinline__ float sb_to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float sb_to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float sb_to_f32<__half>(__half v) { return __half2float(v); }

// Round to nearest even.
template <typename T>
__device__ __forceinline__ T sb_from_f32(float v);
template <>
__device__ __forceinline__ float sb_from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 sb_from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half sb_from_f32<__half>(float v) { return __float2half_rn(v); }

template <typename T, int V>
struct alignas(sizeof(T) * V) SbPack {
  T v[V];
};

template <typename T, int V>
__device__ __forceinline__ SbPack<T, V> sb_load_pack(const T* p) {
  return *reinterpret_cast<const SbPack<T, V>*>(p);
}
// The same as the bytes that were read, where `issue` is set (else `w` keeps what it holds), at this place of the program: an
// ordinary load whose value is used in a branch is moved into that branch by the compiler, and a pack is taken apart right
// behind its load; loads that were to be on their way together then follow one another.  Read-only data, not kept in L1.
template <int BYTES>
struct SbWords;
template <>
struct SbWords<2> { uint16_t v; };
template <>
struct SbWords<4> { uint32_t v; };
template <>
struct SbWords<8> { uint2 v; };
template <>
struct SbWords<16> { uint4 v; };
__device__ __forceinline__ void sb_load_words(SbWords<16>& w, const void* from, bool issue) {
  asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %5, 0;\n\t@q ld.global.nc.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];\n\t}"
               : "+r"(w.v.x), "+r"(w.v.y), "+r"(w.v.z), "+r"(w.v.w) : "l"(from), "r"((uint32_t)issue));
}
__device__ __forceinline__ void sb_load_words(SbWords<8>& w, const void* from, bool issue) {
  asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %3, 0;\n\t@q ld.global.nc.L1::no_allocate.v2.b32 {%0, %1}, [%2];\n\t}"
               : "+r"(w.v.x), "+r"(w.v.y) : "l"(from), "r"((uint32_t)issue));
}
__device__ __forceinline__ void sb_load_words(SbWords<4>& w, const void* from, bool issue) {
  asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %2, 0;\n\t@q ld.global.nc.L1::no_allocate.b32 %0, [%1];\n\t}"
               : "+r"(w.v) : "l"(from), "r"((uint32_t)issue));
}
__device__ __forceinline__ void sb_load_words(SbWords<2>& w, const void* from, bool issue) {
  asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %2, 0;\n\t@q ld.global.nc.L1::no_allocate.b16 %0, [%1];\n\t}"
               : "+h"(w.v) : "l"(from), "r"((uint32_t)issue));
}
// The same, kept in L1 and L2 as an ordinary load is: rows that are read again.
__device__ __forceinline__ void sb_load_kept(SbWords<16>& w, const void* from, bool issue) {
  asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %5, 0;\n\t@q ld.global.nc.v4.b32 {%0, %1, %2, %3}, [%4];\n\t}"
               : "+r"(w.v.x), "+r"(w.v.y), "+r"(w.v.z), "+r"(w.v.w) : "l"(from), "r"((uint32_t)issue));
}
__device__ __forceinline__ void sb_load_kept(SbWords<8>& w, const void* from, bool issue) {
  asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %3, 0;\n\t@q ld.global.nc.v2.b32 {%0, %1}, [%2];\n\t}"
               : "+r"(w.v.x), "+r"(w.v.y) : "l"(from), "r"((uint32_t)issue));
}
__device__ __forceinline__ void sb_load_kept(SbWords<4>& w, const void* from, bool issue) {
  asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %2, 0;\n\t@q ld.global.nc.b32 %0, [%1];\n\t}"
               : "+r"(w.v) : "l"(from), "r"((uint32_t)issue));
}
__device__ __forceinline__ void sb_load_kept(SbWords<2>& w, const void* from, bool issue) {
  asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %2, 0;\n\t@q ld.global.nc.b16 %0, [%1];\n\t}"
               : "+h"(w.v) : "l"(from), "r"((uint32_t)issue));
}
template <typename T, int V>
__device__ __forceinline__ void sb_unpack_words(const SbWords<sizeof(T) * V>& w, float* x) {
  SbPack<T, V> p;
  memcpy(&p, &w, sizeof(p));
#pragma unroll
  for (int i = 0; i < V; ++i) x[i] = sb_to_f32<T>(p.v[i]);
}

template <typename T, int V>
__device__ __forceinline__ SbPack<T, V> sb_zero_pack() {
  SbPack<T, V> r;
#pragma unroll
  for (int i = 0; i < V; ++i) r.v[i] = sb_from_f32<T>(0.f);
  return r;
}
template <typename T, int V>
__device__ __forceinline__ void sb_unpack(const SbPack<T, V>& a, float* x) {
#pragma unroll
  for (int i = 0; i < V; ++i) x[i] = sb_to_f32<T>(a.v[i]);
}
template <typename T, int V>
__device__ __forceinline__ void sb_store_f32(T* p, const float* x) {
  SbPack<T, V> a;
#pragma unroll
  for (int i = 0; i < V; ++i) a.v[i] = sb_from_f32<T>(x[i]);
  *reinterpret_cast<SbPack<T, V>*>(p) = a;
}

// The widest V (a power of two, at most `most`) for which rows that start at `base` with a pitch of `pitch` elements
// and hold `cols` can be taken V elements at a time.
static inline int sb_vector_width(const void* base, long long pitch, long long cols, int item, int most) {
  int v = most;
  while (v > 1 && ((reinterpret_cast<uintptr_t>(base) % (size_t)(v * item)) != 0 || pitch % v != 0 || cols % v != 0)) v /= 2;
  return v;
}
