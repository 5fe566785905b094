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

// One warp per group: the largest magnitude becomes 7 steps.  Single elements and bytes: 4096 x 4096 from fp32 in groups of 128 41 us, where the bytes
// take 12; 512 x 1024 3.2.
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

// A byte per thread: 4096 x 4096 to fp32 38 us, where the bytes take 12.
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

__device__ __forceinline__ void int4_store(const Int4Args& p, long long row, int col, float v, float bias) {
  v += bias;
  if (p.relu) v = fmaxf(v, 0.f);
  const long long at = row * p.ldc + col;
  if (p.out_dtype == SB_F32) reinterpret_cast<float*>(p.c)[at] = v;
  else if (p.out_dtype == SB_BF16) reinterpret_cast<__nv_bfloat16*>(p.c)[at] = __float2bfloat16_rn(v);
  else reinterpret_cast<__half*>(p.c)[at] = __float2half_rn(v);
}

// (w & mask) | bits as one instruction.
__device__ __forceinline__ uint32_t int4_pick(uint32_t w, uint32_t mask, uint32_t bits) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(w), "r"(mask), "r"(bits));
  return r;
}
// Eight codes as four pairs of 16-bit numbers q - 8, (0, 4), (1, 5), (2, 6), (3, 7): with the bits of 1024 (f16) or 128 (bf16) above them a
// code is the number 1024 + q or 128 + q, from which 1032 or 136 is taken without rounding.  Four bits further up, where f16 has room for
// them, it is 1024 + 16 q.  (A common way to unpack whole numbers: it follows from where the formats keep their last bit.)
template <typename T>
__device__ __forceinline__ void int4_pairs(uint32_t w, uint32_t* out) {
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 up = __floats2half2_rn(0.0625f, 0.0625f), low = __floats2half2_rn(-1032.f, -1032.f), high = __floats2half2_rn(-72.f, -72.f);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t a = int4_pick(w, 0x000f000fu, 0x64006400u), b = int4_pick(w, 0x00f000f0u, 0x64006400u);
      const __half2 c = __hadd2(*reinterpret_cast<const __half2*>(&a), low), d = __hfma2(*reinterpret_cast<const __half2*>(&b), up, high);
      memcpy(&out[2 * i], &c, 4);
      memcpy(&out[2 * i + 1], &d, 4);
      w >>= 8;
    }
  } else {
    const __nv_bfloat162 low = __floats2bfloat162_rn(-136.f, -136.f);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t a = int4_pick(w >> (4 * i), 0x000f000fu, 0x43004300u);
      const __nv_bfloat162 c = __hadd2(*reinterpret_cast<const __nv_bfloat162*>(&a), low);
      memcpy(&out[i], &c, 4);
    }
  }
}

struct Int4Few {
  int code_piece;                // bytes of a row of codes that are copied at a time: 16, 8, 4, or 1 where rows start anywhere
  int whole_rows;                // rows of a start on 16 bytes
  int scale_dtype;
  int blocks;                    // of a cluster
  int range;                     // columns of a block, whole steps
  int chunk;                     // of them, those that shared memory holds of a at a time
  int sums_at;                   // where in shared memory the other blocks' sums go
};

// A scale from its 16 bits.
__device__ __forceinline__ float int4_scale(uint32_t bits, int dtype) {
  const float half = __half2float(__ushort_as_half((unsigned short)bits));
  return dtype == SB_BF16 ? __uint_as_float(bits << 16) : half;
}

// N bytes, of which `there` are read and the others zero.
template <int N>
__device__ __forceinline__ void int4_copy(uint32_t to, const void* from, int there) {
  if (N == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(to), "l"(from), "n"(N), "r"(there) : "memory");
}
// Eight elements of a row one by one, `there` of them.
__device__ __noinline__ uint4 int4_elements(const uint16_t* from, int there) {
  uint32_t v[4] = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < there) v[i / 2] |= (uint32_t)from[i] << (16 * (i % 2));
  return make_uint4(v[0], v[1], v[2], v[3]);
}

template <int NT>
constexpr int int4_chunk = NT <= 2 ? 1024 : 2048 / NT;          // columns of a that shared memory holds at most
constexpr int I4_STEP = 256;                            // columns of a stage: 128 bytes of codes a row
constexpr int I4_STAGE = 16 * I4_STEP / 2;
// Where 16 bytes of a row of codes lie in a stage.  The lanes that read together are of two rows and four pieces (groups of 128), of four rows
// and two or of eight and one: with the row's bits in reverse order they meet different banks.
__device__ __forceinline__ uint32_t int4_code_at(int row, int piece) {
  return (uint32_t)(row * 128 + (piece ^ ((row & 1) << 2 | (row & 2) | (row >> 2 & 1))) * 16);
}
// Where eight elements of a row of a (a piece) lie: those of eight rows side by side, turned so that the lanes which read together, of two
// rows and four pieces V apart, meet different banks.
template <int NT, int V>
__device__ __forceinline__ uint32_t int4_at(int piece, int row) {
  return (uint32_t)(((piece * NT + (row >> 3)) * 8 + ((row & 7) ^ (2 * ((piece / V) & 3)))) * 16);
}

// Asks for a stage of a warp's 16 rows, of which `rows` are there with `bytes` bytes, in pieces of PIECE bytes.
template <int PIECE>
__device__ __noinline__ void int4_ask_pieces(uint32_t to, const uint8_t* from, long long pitch, int rows, int bytes) {
  constexpr int ACROSS = 128 / PIECE;
#pragma unroll 4
  for (int e = threadIdx.x & 31; e < 16 * ACROSS; e += 32) {
    const int row = e / ACROSS, b = e % ACROSS * PIECE;
    const int there = row < rows ? min(max(bytes - b, 0), PIECE) : 0;
    const uint32_t at = to + int4_code_at(row, b / 16) + b % 16;
    const uint8_t* source = there > 0 ? from + row * pitch + b : from;
    if constexpr (PIECE >= 4) {
      int4_copy<PIECE>(at, source, there);
    } else {
      const uint16_t v = there > 0 ? *source : (uint16_t)0;
      asm volatile("st.shared.b8 [%0], %1;" ::"r"(at), "h"(v) : "memory");
    }
  }
}

// Asks for a whole stage of 16 rows, each row's 128 bytes by neighbouring lanes.
template <int PIECE>
__device__ __forceinline__ void int4_ask_rows(uint32_t to, const uint8_t* lane_from, long long pitch, int lane) {
  constexpr int ACROSS = 128 / PIECE, DOWN = 32 / ACROSS;
  const int row = lane / ACROSS, b = lane % ACROSS * PIECE;
#pragma unroll
  for (int i = 0; i < 16 / DOWN; ++i, lane_from += DOWN * pitch) int4_copy<PIECE>(to + int4_code_at(row + DOWN * i, b / 16) + b % 16, lane_from, PIECE);
}

__device__ __noinline__ void int4_ask_narrow(uint32_t to, const uint8_t* lane_from, long long pitch, int lane, int piece) {
  if (piece == 8) int4_ask_rows<8>(to, lane_from, pitch, lane);
  else int4_ask_rows<4>(to, lane_from, pitch, lane);
}

// A warp has 16 rows of w, whose codes come to it through a ring of STAGES steps in shared memory; a block's warps share up to 8 NT
// rows of a there, and the blocks of a cluster share K.  The V = G / 32 words of a lane (8 codes each) are of one group in all four lanes
// of a row, so the products of a group are summed as whole numbers times elements of a, and the sums are scaled.  The blocks' sums are
// joined in their order.  Bound by its instructions, 34 per lane and 8 codes for 16 rows of a (nine of them unpack), and by the way to the first and from
// the last of them: 16 x 8192 x 8192 in groups of 64 17.4 us (issue 50 %), where the bytes take 5.5; 1 x 8192 x 8192 in groups of 128 11.  At 128
// registers the forms of 16, 32 and 64 rows of a spill some 10, 50 and 170 bytes a thread.
template <typename T, int G, int NT, int WARPS, int STAGES>
__global__ void __launch_bounds__(32 * WARPS, 16 / WARPS) gemm_int4_kernel(Int4Args p, Int4Few q) {
  constexpr int V = G / 32, PER = I4_STEP / G, COLS = 8 * NT, PITCH = COLS + 2, ROWS = 16 * WARPS;
  extern __shared__ __align__(16) uint8_t i4_smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int blocks = q.blocks, rank = blockIdx.x % blocks;
  const int tile0 = blockIdx.x / blocks * ROWS, r0 = tile0 + 16 * warp, n0 = blockIdx.y * COLS;
  const int begin = min(p.k, rank * q.range), end = min(p.k, begin + q.range);
  uint8_t* ring = i4_smem + warp * (STAGES * I4_STAGE);
  const uint32_t ring_at = smem_u32(ring);
  uint8_t* xs = i4_smem + WARPS * STAGES * I4_STAGE;
  float* scales = reinterpret_cast<float*>(xs + q.chunk * COLS * 2);      // [groups of a chunk][ROWS]
  if (blocks > 1) cluster_arrive_relaxed_all();
  sb_grid_dependency_wait();
  sb_grid_dependents_launch();
  const int steps = (end - begin + I4_STEP - 1) / I4_STEP, groups = (p.k + G - 1) / G, rows = min(16, p.n - r0);
  const int across = 128 / q.code_piece;                                  // lanes that copy a row of a step
  const uint8_t* lane_codes = p.codes + (long long)(r0 + lane / across) * p.ldw + begin / 2 + q.code_piece * (lane % across);
  // Asks for the codes of a step.
  auto ask = [&](int step, int slot) {
    if (step < steps && rows > 0) {
      const int k0 = begin + step * I4_STEP;
      const uint32_t at = ring_at + (uint32_t)(slot * I4_STAGE);
      if (q.code_piece >= 4 && rows == 16 && k0 + I4_STEP <= p.k) {
        const uint8_t* from = lane_codes + step * (I4_STEP / 2);
        if (q.code_piece == 16) int4_ask_rows<16>(at, from, p.ldw, lane);
        else int4_ask_narrow(at, from, p.ldw, lane, q.code_piece);
      } else {
        // What lies beyond k meets zeros of a; rows that are not there are zero.
        const uint8_t* from = p.codes + (long long)r0 * p.ldw + k0 / 2;
        const int bytes = (p.k - k0 + 1) / 2;
        if (q.code_piece == 16) int4_ask_pieces<16>(at, from, p.ldw, rows, bytes);
        else if (q.code_piece == 8) int4_ask_pieces<8>(at, from, p.ldw, rows, bytes);
        else if (q.code_piece == 4) int4_ask_pieces<4>(at, from, p.ldw, rows, bytes);
        else int4_ask_pieces<1>(at, from, p.ldw, rows, bytes);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  // What a chunk needs of a and of the scales is read into registers a chunk ahead: rows of a in the order of the codes' pairs, zeros
  // beyond k and for rows that are not there, of which a thread has one row and every (4 WARPS / NT)-th piece; and the scales of a row of w.
  constexpr int MOST = int4_chunk<NT>, X = MOST / 8 * COLS / (32 * WARPS), SCALES = MOST / G * ROWS / (32 * WARPS);
  const uint16_t* a = reinterpret_cast<const uint16_t*>(p.a);
  const int x_row = threadIdx.x % 8 + threadIdx.x / 32 % NT * 8, x_first = threadIdx.x / 8 % 4 + threadIdx.x / (32 * NT) * 4;
  const int s_row = threadIdx.x % ROWS, s_first = threadIdx.x / ROWS;
  SbWords<16> x_held[X];
  SbWords<2> s_held[SCALES];
  auto load_chunk = [&](int chunk0) {
    const bool there = n0 + x_row < p.m && q.whole_rows;
    const uint16_t* from = a + (long long)(n0 + x_row) * p.lda + chunk0;
#pragma unroll
    for (int i = 0; i < X; ++i) {
      const int at = 8 * (x_first + i * (4 * WARPS / NT));
      x_held[i].v = make_uint4(0u, 0u, 0u, 0u);
      sb_load_kept(x_held[i], from + at, there && at < q.chunk && chunk0 + at + 8 <= p.k);
    }
    const uint16_t* scales_from = reinterpret_cast<const uint16_t*>(p.scales) + (long long)(chunk0 / G) * p.n + tile0 + s_row;
#pragma unroll
    for (int i = 0; i < SCALES; ++i) {
      const int b = s_first + i * (32 * WARPS / ROWS);
      s_held[i].v = 0;
      sb_load_kept(s_held[i], scales_from + (long long)b * p.n, b * G < q.chunk && chunk0 / G + b < groups && tile0 + s_row < p.n);
    }
  };
  auto store_chunk = [&](int chunk0) {
    const uint16_t* from = a + (long long)(n0 + x_row) * p.lda + chunk0;
#pragma unroll
    for (int i = 0; i < X; ++i) {
      const int piece = x_first + i * (4 * WARPS / NT), left = p.k - chunk0 - 8 * piece;
      if (8 * piece >= q.chunk) break;
      uint4 v = x_held[i].v;
      if (n0 + x_row < p.m && left > 0 && (left < 8 || !q.whole_rows)) v = int4_elements(from + 8 * piece, left);
      *reinterpret_cast<uint4*>(xs + int4_at<NT, V>(piece, x_row)) = make_uint4(__byte_perm(v.x, v.z, 0x5410), __byte_perm(v.x, v.z, 0x7632),
                                                                               __byte_perm(v.y, v.w, 0x5410), __byte_perm(v.y, v.w, 0x7632));
    }
#pragma unroll
    for (int i = 0; i < SCALES; ++i) {
      const int b = s_first + i * (32 * WARPS / ROWS);
      if (b * G < q.chunk) scales[b * ROWS + s_row] = int4_scale(s_held[i].v, q.scale_dtype);
    }
  };
  // Before the codes, which are many times more: what everything waits for.
  if (begin < end) load_chunk(begin);
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) ask(s, s);
  // This thread's row of those that this block will finish.
  const int share = ROWS / blocks, out_row = share * rank + threadIdx.x % share;
  const float out_bias = blocks > 1 && p.bias && tile0 + out_row < p.n ? p.bias[tile0 + out_row] : 0.f;

  float acc[NT][4];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[n][j] = 0.f;
  // Where this lane's words lie in a stage (of the group b: with bits of b turned over, eight rows on: 1024 bytes on), and its elements of
  // a in a chunk.
  const uint32_t lane_word = int4_code_at(g, V * t / 4) + 4 * V * t % 16;
  const uint8_t* lane_xs = xs + int4_at<NT, V>(V * t, g);
  int slot = 0, step = 0;
  for (int chunk0 = begin; chunk0 < end; chunk0 += q.chunk) {
    const int chunk1 = min(begin + steps * I4_STEP, chunk0 + q.chunk);
    if (chunk0 != begin) __syncthreads();
    store_chunk(chunk0);
    if (chunk0 + q.chunk < end) load_chunk(chunk0 + q.chunk);
    __syncthreads();
    for (int k0 = chunk0; k0 < chunk1; k0 += I4_STEP, ++step) {
      __syncwarp();                                     // all lanes have read the slot that is filled now
      ask(step + STAGES - 1, slot == 0 ? STAGES - 1 : slot - 1);
      asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
      __syncwarp();
      const uint8_t* stage = ring + slot * I4_STAGE;
      const float* step_scales = scales + (k0 - chunk0) / G * ROWS + 16 * warp + g;
      const uint8_t* step_xs = lane_xs + (k0 - chunk0) / 8 * (NT * 128);
#pragma unroll
      for (int b = 0; b < PER; ++b) {
        SbWords<4 * V> words[2];
        float scale[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          words[h] = *reinterpret_cast<const SbWords<4 * V>*>(stage + (lane_word ^ (uint32_t)(b * (G / 2))) + 1024 * h);
          scale[h] = step_scales[b * ROWS + 8 * h];
        }
        float sum[NT][4];
#pragma unroll
        for (int v = 0; v < V; ++v) {
          uint32_t codes[V], w[2][4];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            memcpy(codes, &words[h], 4 * V);
            int4_pairs<T>(codes[v], w[h]);
          }
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const uint4 x = *reinterpret_cast<const uint4*>(step_xs + ((b * (G / 8) + v) * NT + n) * 128);
            if (v == 0) mma_16x8x16_first<T>(sum[n], w[0][0], w[1][0], w[0][1], w[1][1], x.x, x.y);
            else mma_16x8x16<T>(sum[n], w[0][0], w[1][0], w[0][1], w[1][1], x.x, x.y);
            mma_16x8x16<T>(sum[n], w[0][2], w[1][2], w[0][3], w[1][3], x.z, x.w);
          }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[n][j] = fmaf(scale[j >> 1], sum[n][j], acc[n][j]);
      }
      slot = slot == STAGES - 1 ? 0 : slot + 1;
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  if (blocks == 1) {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int row = r0 + g + 8 * (j >> 1), col = n0 + 8 * n + 2 * t + (j & 1);
        if (row < p.n && col < p.m) int4_store(p, col, row, acc[n][j], p.bias ? p.bias[row] : 0.f);
      }
    return;
  }
  // Each block finishes `share` of the rows: the others lay their sums of these into its shared memory, [blocks][share][PITCH].  All blocks of
  // the cluster have started.
  cluster_wait_all();
  float* sums = reinterpret_cast<float*>(i4_smem + q.sums_at);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int row = 16 * warp + g + 8 * h;
    const uint32_t at = map_to_cta(smem_u32(sums + (rank * share + row % share) * PITCH + 2 * t), (uint32_t)(row / share));
#pragma unroll
    for (int n = 0; n < NT; ++n)
      asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(at + 32u * n), "f"(acc[n][2 * h]), "f"(acc[n][2 * h + 1]) : "memory");
  }
  __syncwarp();
  cluster_sync_all();
  for (int e = threadIdx.x; e < share * COLS; e += 32 * WARPS) {
    const int col = e / share;
    if (tile0 + out_row >= p.n || n0 + col >= p.m) continue;
    float sum = 0.f;
    for (int b = 0; b < blocks; ++b) sum += sums[(b * share + threadIdx.x % share) * PITCH + col];
    int4_store(p, n0 + col, tile0 + out_row, sum, out_bias);
  }
}

// Fewest rows of a (at most 8): a block has 16 rows of w, whose groups its eight warps take in turn, all that a lane needs of UNROLL of
// them on its way to registers at a time and nothing through shared memory but the warps' sums.  Whole groups, codes that start on the
// words of a lane, rows of a that start on 16 bytes.
template <typename T, int G>
__global__ void __launch_bounds__(256, 2) gemm_int4_fewest_kernel(Int4Args p, int scale_dtype) {
  constexpr int V = G / 32, UNROLL = V == 4 ? 2 : 4;
  __shared__ float part[8][16][9];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int r0 = blockIdx.x * 16;
  sb_grid_dependency_wait();
  sb_grid_dependents_launch();
  // Rows that are not there give sums that are not written: they read the last one.
  const int row_a = min(r0 + g, p.n - 1), row_b = min(r0 + g + 8, p.n - 1);
  const uint8_t* codes_a = p.codes + (long long)row_a * p.ldw + 4 * V * t;
  const uint8_t* codes_b = p.codes + (long long)row_b * p.ldw + 4 * V * t;
  const uint16_t* scales = reinterpret_cast<const uint16_t*>(p.scales);
  const T* x = reinterpret_cast<const T*>(p.a) + (long long)g * p.lda + 8 * V * t;
  const bool there = g < p.m;
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  const int groups = p.k / G;
  for (int b0 = warp; b0 < groups; b0 += 8 * UNROLL) {
    SbWords<4 * V> wa[UNROLL], wb[UNROLL];
    SbWords<2> sa[UNROLL], sb[UNROLL];
    SbWords<16> e[UNROLL][V];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int b = b0 + 8 * u;
      const bool in = b < groups;
      memset(&wa[u], 0, 4 * V);
      memset(&wb[u], 0, 4 * V);
      sa[u].v = sb[u].v = 0;
      sb_load_words(wa[u], codes_a + (long long)b * (G / 2), in);
      sb_load_words(wb[u], codes_b + (long long)b * (G / 2), in);
      sb_load_kept(sa[u], scales + (long long)b * p.n + row_a, in);
      sb_load_kept(sb[u], scales + (long long)b * p.n + row_b, in);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        e[u][v].v = make_uint4(0u, 0u, 0u, 0u);
        sb_load_kept(e[u][v], x + b * G + 8 * v, in && there);
      }
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      uint32_t ca[V], cb[V];
      memcpy(ca, &wa[u], 4 * V);
      memcpy(cb, &wb[u], 4 * V);
      float sum[4];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        uint32_t a[4], c[4];
        int4_pairs<T>(ca[v], a);
        int4_pairs<T>(cb[v], c);
        const uint4 y = e[u][v].v;
        const uint32_t x04 = __byte_perm(y.x, y.z, 0x5410), x15 = __byte_perm(y.x, y.z, 0x7632), x26 = __byte_perm(y.y, y.w, 0x5410),
                       x37 = __byte_perm(y.y, y.w, 0x7632);
        if (v == 0) mma_16x8x16_first<T>(sum, a[0], c[0], a[1], c[1], x04, x15);
        else mma_16x8x16<T>(sum, a[0], c[0], a[1], c[1], x04, x15);
        mma_16x8x16<T>(sum, a[2], c[2], a[3], c[3], x26, x37);
      }
      const float scale_a = int4_scale(sa[u].v, scale_dtype), scale_b = int4_scale(sb[u].v, scale_dtype);
      acc[0] = fmaf(scale_a, sum[0], acc[0]);
      acc[1] = fmaf(scale_a, sum[1], acc[1]);
      acc[2] = fmaf(scale_b, sum[2], acc[2]);
      acc[3] = fmaf(scale_b, sum[3], acc[3]);
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) part[warp][g + 8 * (j >> 1)][2 * t + (j & 1)] = acc[j];
  __syncthreads();
  const int row = threadIdx.x % 16, col = threadIdx.x / 16;
  if (col < p.m && r0 + row < p.n) {
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) sum += part[w][row][col];
    int4_store(p, col, r0 + row, sum, p.bias ? p.bias[r0 + row] : 0.f);
  }
}

int int4_args_ok(const char* who, long long n, int k, int group, int scale_dtype) {
  if (n < 0 || k < 0) return sb_fail(SB_ERR_BAD_ARG, "%s: negative size", who);
  if (group != 32 && group != 64 && group != 128) return sb_fail(SB_ERR_UNSUPPORTED, "%s: groups of 32, 64 or 128 (got %d)", who, group);
  if (scale_dtype != SB_BF16 && scale_dtype != SB_F16) return sb_fail(SB_ERR_UNSUPPORTED, "%s: scales are bf16 or f16 (got %d)", who, scale_dtype);
  if (n > (1LL << 30) || k > (1 << 30)) return sb_fail(SB_ERR_TOO_LARGE, "%s: at most 2^30 rows and columns", who);
  return SB_OK;
}

bool int4_aligned(const void* p, int dtype) { return reinterpret_cast<uintptr_t>(p) % (size_t)sb_dtype_size(dtype) == 0; }

// The form of a product: rows of a that a block has (0: the fewest, straight to registers), and blocks that share K.
struct Int4Form {
  int rows, blocks;
};
Int4Form int4_form(long long m, long long n, int k, int group, int code_piece, bool whole_rows) {
  const long long sms = sb_sm_count();
  // Small matrices of weights, whose time is that of the way there: 1 x 4096 x 4096 in groups of 128 4.8 us, through rings 6.1; 1 x 256 x 512
  // 2.1 / 4.5; 8 x 4096 x 4096 6.5 / 6.5.  Not long rows (1 x 1024 x 16384 27 / 12) nor more blocks than there is room for (1 x 8192 x 8192
  // 17.5 / 14.2).
  if (m <= 8 && k <= 4096 && n <= 32 * sms && k % group == 0 && code_piece >= group / 8 && whole_rows) return {0, 1};
  // Where all blocks run at once (or, of 16 rows, nearly), fewer rows of a in each and more blocks: 48 x 201 x 12728 with 64 / 16 / 8 rows of a in a
  // block 53 / 20.5 / 12.2 us, 64 x 1024 x 1024 15.1 / 6.5 / 5.6, 64 x 2048 x 2048 15.6 / 8.0 / 8.8, 64 x 4096 x 4096 32 / 18.6 / 23, 16 x 3000 x 6000
  // 9.9 (16) / 14.1.  At the rule's border 32 x 8192 x 8192 with 32 / 16 / 8 rows takes 32.5 / 32.3 / 49, behind it 48 x 8192 x 8192 with 64 / 16 58 / 60.
  const long long shares = k >= 2048 ? 8 : k >= 1024 ? 4 : k >= 512 ? 2 : 1;
  int rows = m <= 32 ? 32 : 64;
  if (m <= 8 || (n + 127) / 128 * ((m + 7) / 8) * shares <= 2 * sms) rows = 8;
  else if (m <= 16 || (n + 255) / 256 * ((m + 15) / 16) * shares <= 4 * sms) rows = 16;
  // Blocks that share K until every SM has the warps it can hold, each with 256 columns at least.
  const int warps = rows == 8 ? 8 : 16;
  const long long tiles = (n + 16 * warps - 1) / (16 * warps), down = (m + rows - 1) / rows;
  int blocks = 1;
  // Not in clusters of 8 that the chip's parts have no room for at once: 16 x 4096 x 4096 in 16 of them 14.5 us, in clusters of 4 10.4.
  const long long room = (16 / warps) * sms, room8 = warps == 16 ? 3 * room / 4 : 7 * room / 8;
  while (blocks < 8 && tiles * down * blocks * 2 <= (blocks < 4 ? room : room8) && k >= 512 * blocks) blocks *= 2;
  return {rows, blocks};
}

template <typename T, int G, int NT, int WARPS, int STAGES>
int launch_int4(const Int4Args& p, Int4Few q, int blocks, cudaStream_t s) {
  constexpr int ROWS = 16 * WARPS, COLS = 8 * NT, MOST = int4_chunk<NT>, RING = WARPS * STAGES * I4_STAGE, SUMS = ROWS * (COLS + 2) * 4, LIMIT = RING + MOST * COLS * 2 + MOST / G * ROWS * 4 + SUMS;
  static_assert(LIMIT <= 227 * 1024, "more shared memory than an SM has");
  const long long tiles = ((long long)p.n + ROWS - 1) / ROWS, down = ((long long)p.m + COLS - 1) / COLS;
  q.blocks = blocks;
  q.range = ((p.k + blocks - 1) / blocks + I4_STEP - 1) / I4_STEP * I4_STEP;
  q.chunk = q.range < MOST ? q.range : MOST;
  q.sums_at = RING + q.chunk * COLS * 2 + q.chunk / G * ROWS * 4;
  const int bytes = q.sums_at + (blocks > 1 ? SUMS : 0);
  static std::atomic<bool> ready[64];
  const int rc = sb_allow_smem(gemm_int4_kernel<T, G, NT, WARPS, STAGES>, LIMIT, ready);
  if (rc != SB_OK) return rc;
  SB_CUDA(sb_launch(gemm_int4_kernel<T, G, NT, WARPS, STAGES>, dim3((unsigned)(tiles * blocks), (unsigned)down), dim3(32 * WARPS), (size_t)bytes, s, blocks, p, q));
  SB_COUNT_LAUNCH();
  return SB_OK;
}

template <typename T, int G>
int launch_int4(const Int4Args& p, const Int4Few& q, cudaStream_t s) {
  const Int4Form form = int4_form(p.m, p.n, p.k, G, q.code_piece, q.whole_rows != 0);
  if (form.rows == 0) {
    SB_CUDA(sb_launch(gemm_int4_fewest_kernel<T, G>, dim3((unsigned)(((long long)p.n + 15) / 16)), dim3(256), 0, s, 1, p, q.scale_dtype));
    SB_COUNT_LAUNCH();
    return SB_OK;
  }
  if (form.rows == 8) return launch_int4<T, G, 1, 8, 4>(p, q, form.blocks, s);
  if (form.rows == 16) return launch_int4<T, G, 2, 16, 4>(p, q, form.blocks, s);
  if (form.rows == 32) return launch_int4<T, G, 4, 16, 4>(p, q, form.blocks, s);
  return launch_int4<T, G, 8, 16, 3>(p, q, form.blocks, s);
}

// The widest pieces in which rows can be copied.
int int4_piece(const void* p, long long pitch, int least) {
  for (int piece = 16; piece >= 4; piece /= 2)
    if (reinterpret_cast<uintptr_t>(p) % piece == 0 && pitch % piece == 0) return piece;
  return least;
}

template <typename T>
int launch_int4(const Int4Args& p, int scale_dtype, cudaStream_t s) {
  Int4Few q;
  memset(&q, 0, sizeof(q));
  q.code_piece = int4_piece(p.codes, p.n == 1 ? 16 : p.ldw, 1);
  q.whole_rows = int4_piece(p.a, p.m == 1 ? 16 : 2 * p.lda, 2) == 16 ? 1 : 0;
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
  if ((const void*)codes == x || scales == x || scales == (const void*)codes) return sb_fail(SB_ERR_BAD_ARG, "%s: codes and scales have places of their own", who);
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
  if (out == (const void*)codes || out == scales) return sb_fail(SB_ERR_BAD_ARG, "%s: the output in the place of codes or scales", who);
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
  if (k > 0 && (c == a || c == (const void*)codes || c == scales)) return sb_fail(SB_ERR_BAD_ARG, "%s: c in the place of what it is made from", who);
  if ((epilogue & SB_EPI_BIAS) && c == (const void*)bias) return sb_fail(SB_ERR_BAD_ARG, "%s: c in the place of the bias", who);
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

int sb_matmul_int4_plan(int m, int n, int k, int group, int* plan) {
  const char* who = "sb_matmul_int4_plan";
  int rc = int4_args_ok(who, n, k, group, SB_BF16);
  if (rc != SB_OK) return rc;
  if (!plan) return sb_fail(SB_ERR_BAD_ARG, "%s: null output", who);
  if (m <= 0 || n == 0 || k == 0) return sb_fail(SB_ERR_BAD_ARG, "%s: sizes of nothing", who);
  const Int4Form form = int4_form(m, n, k, group, int4_piece(nullptr, n == 1 ? 16 : (k + 1) / 2, 1), int4_piece(nullptr, m == 1 ? 16 : 2LL * k, 2) == 16);
  plan[0] = form.rows;
  plan[1] = form.blocks;
  return SB_OK;
}

}  // extern "C"
