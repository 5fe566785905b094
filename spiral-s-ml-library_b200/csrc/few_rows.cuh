// Products of few rows with weights that are read once, as warp-level matrix instructions on operands that go from memory to
// registers: 16 weight rows are the instruction's rows, 8 rows of the activations its columns.  Memory bound: a weight of 16
// bits takes part in at most 16 rows' products, where tcgen05 would need 128 and a trip through shared memory.
//
// The order of K within an instruction is free as long as both operands share it: lane (g, t) = (lane / 4, lane % 4) takes eight
// neighbouring elements of a row at 8 t, one 16-byte load, as its fragments of two instructions of 16.
#pragma once

#include "common.cuh"
#include "vector_io.cuh"

// c[16 x 8] += a[16 x 16] b[16 x 8]: a0 and a2 are of row g, a1 and a3 of row g + 8; c0, c1 are columns 2 t, 2 t + 1 of row g, c2, c3 of row
// g + 8.
template <typename T>
__device__ __forceinline__ void mma_16x8x16(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma_16x8x16<__nv_bfloat16>(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma_16x8x16<__half>(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The same with c = 0 before.
template <typename T>
__device__ __forceinline__ void mma_16x8x16_first(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma_16x8x16_first<__nv_bfloat16>(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
               : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
template <>
__device__ __forceinline__ void mma_16x8x16_first<__half>(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
               : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

// Eight 16-bit elements from column k0 on of a row that holds `k`, zeros beyond and for rows that are not there: one load, but for
// the row's last ones.  `row` + k0 is 16-byte aligned.  KEPT: rows that are read again.
template <bool KEPT>
__device__ __forceinline__ uint4 load_eight(const void* row, long long k0, long long k, bool there) {
  SbWords<16> w;
  w.v = make_uint4(0u, 0u, 0u, 0u);
  const uint16_t* p = reinterpret_cast<const uint16_t*>(row) + k0;
  const bool whole = there && k0 + 8 <= k;
  if (KEPT) sb_load_kept(w, p, whole);
  else sb_load_words(w, p, whole);
  if (there && !whole && k0 < k) {
    uint32_t v[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int i = 0; i < 7; ++i)
      if (k0 + i < k) v[i / 2] |= (uint32_t)p[i] << (16 * (i % 2));
    w.v = make_uint4(v[0], v[1], v[2], v[3]);
  }
  return w.v;
}
