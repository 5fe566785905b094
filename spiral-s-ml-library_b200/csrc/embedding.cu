// Embedding lookup with scaling, and its gradient by sorted tokens.
//
//   out[i, :] = scale * table[t_i, :]                       a token outside [0, vocab) gives a row of zeros
//   dtable[v, :] = scale * sum over i with t_i = v of dout[i, :]   (+ the old values when accumulating)
//
// The gradient adds each token's rows in the order of their positions: the tokens are sorted (stable radix sort of
// (token, position) pairs), and the sorted list and the rows of the table are walked together, cut into runs of equal
// length (rows read + rows written), so that neither a token that fills half of the batch nor a vocabulary that is
// mostly absent leaves anybody without work.  A token whose positions span several runs leaves a partial sum behind
// each; a last kernel adds those in the order of the runs.  Sums are fp32, without atomics: two calls give the same bits.
#include "common.cuh"
#include "vector_io.cuh"

namespace {

// ------------------------------- lookup -----------------------------------------
// A thread per V neighbouring elements of the output.  Tables are stored with a row pitch.
template <typename I, typename T, typename O, int V>
__global__ void __launch_bounds__(256)
embedding_kernel(const I* __restrict__ tokens, const T* __restrict__ table, O* __restrict__ out, long long n, int vocab, int dim,
                 long long ld_table, long long ld_out, float scale) {
  sb_grid_dependency_wait();
  sb_grid_dependents_launch();
  const int pieces = dim / V;
  const long long total = n * pieces, step = (long long)gridDim.x * blockDim.x;
  for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += step) {
    const long long r = i / pieces;
    const int c = (int)(i - r * pieces) * V;
    const long long t = (long long)tokens[r];
    float v[V];
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = 0.f;
    if (t >= 0 && t < vocab) {
      sb_unpack<T, V>(sb_load_pack<T, V>(table + t * ld_table + c), v);
#pragma unroll
      for (int k = 0; k < V; ++k) v[k] *= scale;
    }
    sb_store_f32<O, V>(out + r * ld_out + c, v);
  }
}

// -------------------------------- sort ------------------------------------------
constexpr int ES_THREADS = 256;
constexpr int ES_WARPS = ES_THREADS / 32;
constexpr int ES_MAX_BITS = 11;
constexpr int ES_MAX_BINS = 1 << ES_MAX_BITS;

struct SortPlan {
  int passes, bits;              // digits, and bits of each
  int rounds;                    // tokens per thread of a chunk
  int chunk, chunks;
};

// Digits of at most 11 bits, all of one size, that together cover the keys 0 .. vocab (vocab: no token).
SortPlan sort_plan(long long n, int vocab) {
  SortPlan p;
  int bits = 1;
  while (bits < 31 && (1LL << bits) <= vocab) ++bits;
  p.passes = (bits + ES_MAX_BITS - 1) / ES_MAX_BITS;
  p.bits = (bits + p.passes - 1) / p.passes;
  // Chunks of 1024 tokens until there are several per SM, then of 4096.
  p.rounds = n > 1024LL * 4 * sb_sm_count() ? 16 : 4;
  p.chunk = ES_THREADS * p.rounds;
  p.chunks = (int)((n + p.chunk - 1) / p.chunk);
  return p;
}

struct SortArgs {
  const void* tokens;            // first pass: the caller's tokens (int32 or int64)
  const int* keys_in;            // later passes
  const int* pos_in;
  int* keys_out;
  int* pos_out;
  int* counts;                   // [bins][chunks], turned into the bin's running sums by the scan
  int* totals;                   // [bins]
  int n, vocab, shift, bits, chunks, chunk;
  int index64;
};

template <bool FIRST>
__device__ __forceinline__ int sort_key(const SortArgs& a, int i) {
  if (!FIRST) return a.keys_in[i];
  const long long t = a.index64 ? ((const long long*)a.tokens)[i] : (long long)((const int*)a.tokens)[i];
  return t >= 0 && t < a.vocab ? (int)t : a.vocab;
}

template <bool FIRST>
__global__ void __launch_bounds__(ES_THREADS) token_count_kernel(SortArgs a) {
  __shared__ int hist[ES_MAX_BINS];
  const int bins = 1 << a.bits;
  for (int b = threadIdx.x; b < bins; b += ES_THREADS) hist[b] = 0;
  sb_grid_dependency_wait();
  sb_grid_dependents_launch();
  __syncthreads();
  // Equal digits of a warp are added as one: with the 53 tokens of a deck most lanes of a warp meet in a few words.
  const int first = blockIdx.x * a.chunk, last = min(a.n - first, a.chunk) + first;
  for (int i0 = first; i0 < last; i0 += ES_THREADS) {
    const int i = i0 + threadIdx.x;
    const int digit = i < last ? (sort_key<FIRST>(a, i) >> a.shift) & (bins - 1) : bins;
    const unsigned same = __match_any_sync(0xffffffffu, digit);
    if (digit < bins && (same & ((1u << (threadIdx.x & 31)) - 1u)) == 0u) atomicAdd(&hist[digit], __popc(same));
  }
  __syncthreads();
  for (int b = threadIdx.x; b < bins; b += ES_THREADS) a.counts[(long long)b * a.chunks + blockIdx.x] = hist[b];
}

__device__ __forceinline__ int warp_inclusive(int v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += up;
  }
  return v;
}

// A warp per bin: running sums of its counts over the chunks, and its total.
__global__ void __launch_bounds__(256) token_scan_kernel(SortArgs a) {
  sb_grid_dependency_wait();
  sb_grid_dependents_launch();
  const int bin = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (bin >= (1 << a.bits)) return;
  int* c = a.counts + (long long)bin * a.chunks;
  int before = 0;
  for (int i0 = 0; i0 < a.chunks; i0 += 32) {
    const int v = i0 + lane < a.chunks ? c[i0 + lane] : 0;
    const int up = warp_inclusive(v);
    if (i0 + lane < a.chunks) c[i0 + lane] = before + up - v;
    before += __shfl_sync(0xffffffffu, up, 31);
  }
  if (lane == 0) a.totals[bin] = before;
}

// Puts a chunk's (token, position) pairs where they belong by this digit, those of equal digits in their order: a warp
// takes a run of consecutive tokens 32 at a time; equal digits within the 32 find each other by a match.
template <bool FIRST, int ROUNDS>
__global__ void __launch_bounds__(ES_THREADS) token_scatter_kernel(SortArgs a) {
  extern __shared__ int s_scatter[];
  const int bins = 1 << a.bits;
  int* base = s_scatter;                                     // [bins]: where the chunk's first token of the bin goes
  unsigned short* seen = reinterpret_cast<unsigned short*>(s_scatter + bins);   // [warps][bins]
  __shared__ int warp_total[ES_WARPS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int b = threadIdx.x; b < bins * ES_WARPS; b += ES_THREADS) seen[b] = 0;
  sb_grid_dependency_wait();
  sb_grid_dependents_launch();
  // Exclusive sums of the bins' totals: each thread a run of bins.
  const int per = (bins + ES_THREADS - 1) / ES_THREADS;
  int mine = 0;
  for (int k = 0; k < per; ++k) {
    const int b = threadIdx.x * per + k;
    if (b < bins) mine += a.totals[b];
  }
  const int incl = warp_inclusive(mine);
  if (lane == 31) warp_total[warp] = incl;
  __syncthreads();
  int run = incl - mine;
  for (int w = 0; w < warp; ++w) run += warp_total[w];
  for (int k = 0; k < per; ++k) {
    const int b = threadIdx.x * per + k;
    if (b < bins) {
      base[b] = run + a.counts[(long long)b * a.chunks + blockIdx.x];
      run += a.totals[b];
    }
  }
  const int first = blockIdx.x * a.chunk + warp * (32 * ROUNDS);
  int key[ROUNDS];
  unsigned short rank[ROUNDS];
  unsigned short* mine_seen = seen + warp * bins;
#pragma unroll
  for (int k = 0; k < ROUNDS; ++k) {
    const int i = first + k * 32 + lane;
    key[k] = i >= 0 && i < a.n ? sort_key<FIRST>(a, i) : -1;
  }
#pragma unroll
  for (int k = 0; k < ROUNDS; ++k) {
    const int digit = key[k] < 0 ? bins : (key[k] >> a.shift) & (bins - 1);
    const unsigned same = __match_any_sync(0xffffffffu, digit);
    const int before = __popc(same & ((1u << lane) - 1u));
    if (digit < bins) rank[k] = (unsigned short)(mine_seen[digit] + before);
    __syncwarp();
    if (digit < bins && before == 0) mine_seen[digit] = (unsigned short)(mine_seen[digit] + __popc(same));
    __syncwarp();
  }
  __syncthreads();
  for (int b = threadIdx.x; b < bins; b += ES_THREADS) {
    int at = 0;
#pragma unroll
    for (int w = 0; w < ES_WARPS; ++w) {
      const int c = seen[w * bins + b];
      seen[w * bins + b] = (unsigned short)at;
      at += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < ROUNDS; ++k) {
    if (key[k] < 0) continue;
    const int i = first + k * 32 + lane;
    const int digit = (key[k] >> a.shift) & (bins - 1);
    const int to = base[digit] + mine_seen[digit] + rank[k];
    a.keys_out[to] = key[k];
    a.pos_out[to] = FIRST ? i : a.pos_in[i];
  }
}

// Up to ES_SMALL tokens: one block sorts them in shared memory, 8 bits at a time.
constexpr int ES_SMALL = 4096;
constexpr int ES_SMALL_THREADS = 1024;
__global__ void __launch_bounds__(ES_SMALL_THREADS) token_sort_small_kernel(SortArgs a, int bits) {
  constexpr int BINS = 256, WARPS = ES_SMALL_THREADS / 32, ROUNDS = ES_SMALL / ES_SMALL_THREADS;
  extern __shared__ int s_sort[];
  int* keys = s_sort;
  unsigned short* pos = reinterpret_cast<unsigned short*>(keys + ES_SMALL);
  unsigned short* seen = pos + ES_SMALL;                     // [warps][bins]
  __shared__ int base[BINS], warp_total[BINS / 32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  sb_grid_dependency_wait();
  sb_grid_dependents_launch();
  int key[ROUNDS], at[ROUNDS];
#pragma unroll
  for (int k = 0; k < ROUNDS; ++k) {
    at[k] = warp * (32 * ROUNDS) + k * 32 + lane;
    key[k] = at[k] < a.n ? sort_key<true>(a, at[k]) : -1;
  }
  for (int shift = 0; shift < bits; shift += 8) {
    for (int b = threadIdx.x; b < BINS * WARPS / 2; b += ES_SMALL_THREADS) reinterpret_cast<int*>(seen)[b] = 0;
    __syncthreads();
    unsigned short rank[ROUNDS];
    unsigned short* mine = seen + warp * BINS;
#pragma unroll
    for (int k = 0; k < ROUNDS; ++k) {
      const int digit = key[k] < 0 ? BINS : (key[k] >> shift) & (BINS - 1);
      const unsigned same = __match_any_sync(0xffffffffu, digit);
      const int before = __popc(same & ((1u << lane) - 1u));
      if (digit < BINS) rank[k] = (unsigned short)(mine[digit] + before);
      __syncwarp();
      if (digit < BINS && before == 0) mine[digit] = (unsigned short)(mine[digit] + __popc(same));
      __syncwarp();
    }
    __syncthreads();
    int total = 0, incl = 0;
    if (threadIdx.x < BINS) {
#pragma unroll 8
      for (int w = 0; w < WARPS; ++w) {
        const int c = seen[w * BINS + threadIdx.x];
        seen[w * BINS + threadIdx.x] = (unsigned short)total;
        total += c;
      }
      incl = warp_inclusive(total);
      if (lane == 31) warp_total[warp] = incl;
    }
    __syncthreads();
    if (threadIdx.x < BINS) {
      int run = incl - total;
      for (int w = 0; w < warp; ++w) run += warp_total[w];
      base[threadIdx.x] = run;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < ROUNDS; ++k)
      if (key[k] >= 0) {
        const int digit = (key[k] >> shift) & (BINS - 1), to = base[digit] + mine[digit] + rank[k];
        keys[to] = key[k];
        pos[to] = (unsigned short)at[k];
      }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < ROUNDS; ++k) {
      const int i = warp * (32 * ROUNDS) + k * 32 + lane;
      key[k] = i < a.n ? keys[i] : -1;
      at[k] = i < a.n ? pos[i] : 0;
    }
  }
#pragma unroll
  for (int k = 0; k < ROUNDS; ++k) {
    const int i = warp * (32 * ROUNDS) + k * 32 + lane;
    if (i < a.n) {
      a.keys_out[i] = key[k];
      a.pos_out[i] = at[k];
    }
  }
}

// ------------------------------ gradient ----------------------------------------
struct GradArgs {
  const int* keys;               // sorted tokens (vocab: none)
  const int* pos;
  const void* dout;
  float* dtable;
  float* carry;                  // [runs][dim]: what a run adds to the row that it leaves unfinished
  int* run_key;                  // [runs + 1]: tokens consumed where a run begins
  long long ld_dout, ld_dtable;
  int n, vocab, dim;
  int run_len, runs;             // steps (rows read + rows written) per run
  int group;                     // threads that share a run
  float scale;
  int accumulate;
};

// The walk over sorted tokens and table rows: after d steps k tokens have been added and d - k rows finished, where a
// row is finished when all tokens up to it have been added.  A warp looks for k, 32 places at a time.
__device__ __forceinline__ int walk_split(const int* __restrict__ keys, int n, int vocab, long long d) {
  long long lo = d > vocab ? d - vocab : 0, hi = d < n ? d : n;
  while (lo < hi) {
    const long long step = (hi - lo + 31) / 32, at = lo + (threadIdx.x & 31) * step;
    const bool before = at < hi && (long long)keys[at] <= d - 1 - at;      // true up to the place looked for
    const int count = __popc(__ballot_sync(0xffffffffu, before));
    if (count == 0) {
      hi = lo;
    } else {
      hi = min(hi, lo + count * step);
      lo = lo + (count - 1) * step + 1;
    }
  }
  return (int)lo;
}

// The rows that a block adds up and finishes: groups x run_len steps of the walk, whose tokens and positions it brings to
// shared memory; a group of threads per run, V neighbouring columns per thread, the next UNROLL rows of dout on their way
// while the ones before are added.  (Every group searching the sorted tokens for itself, 17 dependent loads twice, and
// reading token and position from global memory in the loop: 50001 x 1000 fp32 213 us.)
template <typename T, int V>
__global__ void __launch_bounds__(256) embedding_grad_kernel(GradArgs a) {
  constexpr int UNROLL = 8;
  extern __shared__ int s_walk[];
  __shared__ int ends[2];
  const int groups = blockDim.x / a.group;
  const int steps = groups * a.run_len;
  int* s_key = s_walk;
  int* s_pos = s_walk + steps;
  const long long first = (long long)blockIdx.x * steps, all = (long long)a.n + a.vocab;
  sb_grid_dependency_wait();
  sb_grid_dependents_launch();
  if (threadIdx.x < 64) {
    const int which = threadIdx.x >> 5;
    const int k = walk_split(a.keys, a.n, a.vocab, which == 0 ? first : min(first + steps, all));
    if ((threadIdx.x & 31) == 0) ends[which] = k;
  }
  __syncthreads();
  const int k_first = ends[0], count = ends[1] - k_first;
  for (int i = threadIdx.x; i < count; i += blockDim.x) {
    s_key[i] = a.keys[k_first + i];
    s_pos[i] = a.pos[k_first + i];
  }
  __syncthreads();
  const int in_group = threadIdx.x % a.group;
  const int run = blockIdx.x * groups + threadIdx.x / a.group;
  const int col = (blockIdx.y * a.group + in_group) * V;
  if (run >= a.runs) return;
  // The run's own part, by halves.
  auto split = [&](long long d) {
    int lo = (int)max(0LL, d - a.vocab - k_first), hi = (int)min((long long)count, d - k_first);
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if ((long long)s_key[mid] <= d - 1 - (k_first + mid)) lo = mid + 1;
      else hi = mid;
    }
    return lo;
  };
  const long long d0 = (long long)run * a.run_len, d1 = min(d0 + a.run_len, all);
  int k = split(d0);
  const int k_end = split(d1);
  if (blockIdx.y == 0 && in_group == 0) {
    a.run_key[run] = k_first + k;
    if (run == a.runs - 1) a.run_key[a.runs] = k_first + k_end;
  }
  if (col >= a.dim) return;
  int row = (int)(d0 - (k_first + k));
  const int row_end = (int)(d1 - (k_first + k_end));
  const T* dout = (const T*)a.dout + col;
  float* to = a.dtable + (long long)row * a.ld_dtable + col;
  float acc[V];
#pragma unroll
  for (int t = 0; t < V; ++t) acc[t] = 0.f;
  auto finish = [&]() {
    float out[V];
#pragma unroll
    for (int t = 0; t < V; ++t) out[t] = acc[t] * a.scale;
    if (a.accumulate) {
#pragma unroll
      for (int t = 0; t < V; ++t) out[t] += to[t];
    }
#pragma unroll
    for (int t = 0; t < V; t += 4) {
      if constexpr (V >= 4) sb_store_f32<float, 4>(to + t, out + t);
      else sb_store_f32<float, V>(to, out);
    }
#pragma unroll
    for (int t = 0; t < V; ++t) acc[t] = 0.f;
    to += a.ld_dtable;
    ++row;
  };
  while (k < k_end) {
    SbPack<T, V> in[UNROLL];
    int key[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      key[u] = k + u < k_end ? s_key[k + u] : a.vocab;
      if (key[u] < a.vocab) in[u] = sb_load_pack<T, V>(dout + (long long)s_pos[k + u] * a.ld_dout);
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      if (key[u] < a.vocab) {
        while (row < key[u]) finish();
        float v[V];
        sb_unpack<T, V>(in[u], v);
#pragma unroll
        for (int t = 0; t < V; ++t) acc[t] += v[t];
      }
    }
    k += UNROLL;
  }
  while (row < row_end) finish();
  float* carry = a.carry + (long long)run * a.dim + col;
#pragma unroll
  for (int t = 0; t < V; ++t) carry[t] = acc[t];
}

// A table of few rows needs no sort: every warp (or part of one) adds its share of the positions, in their order, to a table of
// its own in shared memory, V columns per thread and G x V per block; the block adds its tables up, and the blocks' sums are
// added in their order by a second launch.  Bound by reading dout: 524288 x 64 bf16 over 53 tokens, PLACEHOLDER.
constexpr int EF_THREADS = 512;
constexpr int EF_SMEM = 200 * 1024;
struct FewArgs {
  const void* tokens;
  const void* dout;
  float* dtable;                 // written directly by a single block
  float* partial;                // [blocks][vocab][dim], else
  long long ld_dout, ld_dtable;
  int n, vocab, dim, index64;
  int lanes, copies;             // threads per position; tables per block
  int per;                       // positions per table
  float scale;
  int accumulate;
};

template <typename T, int V>
__global__ void __launch_bounds__(EF_THREADS) embedding_few_kernel(FewArgs a) {
  constexpr int UNROLL = 8;
  extern __shared__ __align__(16) float s_tables[];          // [copies][vocab][lanes * V]
  const int width = a.lanes * V, table = a.vocab * width;
  const int copy = threadIdx.x / a.lanes, lane = threadIdx.x % a.lanes;
  for (int i = threadIdx.x; i < a.copies * table; i += blockDim.x) s_tables[i] = 0.f;
  sb_grid_dependency_wait();
  sb_grid_dependents_launch();
  __syncthreads();
  const int col = (blockIdx.y * a.lanes + lane) * V;
  const long long first = ((long long)blockIdx.x * a.copies + copy) * a.per;
  const int count = (int)max(0LL, min((long long)a.per, a.n - first));
  if (copy < a.copies && col < a.dim) {
    float* mine = s_tables + copy * table + lane * V;
    const T* dout = (const T*)a.dout + first * a.ld_dout + col;
    for (int i = 0; i < count; i += UNROLL) {
      SbPack<T, V> in[UNROLL];
      int token[UNROLL];
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) {
        token[u] = -1;
        if (i + u < count) {
          const long long t = a.index64 ? ((const long long*)a.tokens)[first + i + u] : (long long)((const int*)a.tokens)[first + i + u];
          if (t >= 0 && t < a.vocab) token[u] = (int)t;
        }
      }
#pragma unroll
      for (int u = 0; u < UNROLL; ++u)
        if (token[u] >= 0) in[u] = sb_load_pack<T, V>(dout + u * a.ld_dout);
#pragma unroll
      for (int u = 0; u < UNROLL; ++u)
        if (token[u] >= 0) {
          float v[V], t[V];
          sb_unpack<T, V>(in[u], v);
          float* to = mine + token[u] * width;
          sb_unpack<float, V>(sb_load_pack<float, V>(to), t);
#pragma unroll
          for (int k = 0; k < V; ++k) t[k] += v[k];
          sb_store_f32<float, V>(to, t);
        }
      dout += UNROLL * a.ld_dout;
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < table; i += blockDim.x) {
    const int row = i / width, c = blockIdx.y * width + i % width;
    if (c >= a.dim) continue;
    float total = 0.f;
    for (int k = 0; k < a.copies; ++k) total += s_tables[k * table + i];
    if (gridDim.x == 1) {
      float* to = a.dtable + row * a.ld_dtable + c;
      *to = a.accumulate ? *to + total * a.scale : total * a.scale;
    } else {
      a.partial[((long long)blockIdx.x * a.vocab + row) * a.dim + c] = total;
    }
  }
}

// The blocks' sums in their order: 32 neighbouring elements per block, its warps take every 32nd part.
__global__ void __launch_bounds__(1024) embedding_few_join_kernel(FewArgs a, int parts) {
  __shared__ float sums[32][33];
  sb_grid_dependency_wait();
  sb_grid_dependents_launch();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long size = (long long)a.vocab * a.dim, i = (long long)blockIdx.x * 32 + lane;
  float s = 0.f;
  if (i < size)
    for (int p = warp; p < parts; p += 32) s += a.partial[p * size + i];
  sums[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && i < size) {
    float total = 0.f;
#pragma unroll
    for (int w = 0; w < 32; ++w) total += sums[w][lane];
    float* to = a.dtable + i / a.dim * a.ld_dtable + i % a.dim;
    *to = a.accumulate ? *to + total * a.scale : total * a.scale;
  }
}

// Adds what runs left unfinished to the row that a later run finished: a block of 8 warps per such run and 32 columns; every
// warp takes a part of the runs before it, in order, and the warps' sums meet in shared memory.
__global__ void __launch_bounds__(256) embedding_join_kernel(GradArgs a) {
  __shared__ float sums[8][32];
  sb_grid_dependency_wait();
  sb_grid_dependents_launch();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long all = (long long)a.n + a.vocab;
  for (int run = blockIdx.x + 1; run < a.runs; run += gridDim.x) {
    const long long d0 = (long long)run * a.run_len, d1 = min(d0 + a.run_len, all);
    const int k0 = a.run_key[run], row = (int)(d0 - k0), row_end = (int)(d1 - a.run_key[run + 1]);
    // Only where this run finishes a row that tokens of earlier runs have been added to.
    if (row >= a.vocab || row_end == row || k0 == 0 || a.keys[k0 - 1] != row) continue;
    int lo = 0, hi = run;        // the first run that ends in this row
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if ((long long)(mid + 1) * a.run_len - a.run_key[mid + 1] >= row) hi = mid;
      else lo = mid + 1;
    }
    const int parts = run - lo, per = (parts + 7) / 8;
    const int from = lo + warp * per, to = min(run, from + per);
    for (int c = blockIdx.y * 32 + lane; c < (a.dim + 31) / 32 * 32; c += 32 * gridDim.y) {
      float s = 0.f;
      if (c < a.dim) {
#pragma unroll 4
        for (int r = from; r < to; ++r) s += a.carry[(long long)r * a.dim + c];
      }
      sums[warp][lane] = s;
      __syncthreads();
      if (warp == 0 && c < a.dim) {
        float total = 0.f;
#pragma unroll
        for (int w = 0; w < 8; ++w) total += sums[w][lane];
        a.dtable[(long long)row * a.ld_dtable + c] += total * a.scale;
      }
      __syncthreads();
    }
  }
}

struct FewPlan {
  int v, lanes, copies, per, blocks, slabs;
};

// A table of at most 100 rows or so: six or more copies of 64 columns (two per thread; 32 or fewer, one per thread, where dout does not
// allow pairs) fit into a block's shared memory.
bool few_plan(long long n, int vocab, int dim, int v, FewPlan* p) {
  p->v = dim >= 64 ? v : 1;
  p->lanes = 32;
  if (p->v == 1)
    while (p->lanes > 4 && p->lanes / 2 >= dim) p->lanes /= 2;
  const long long table = 4LL * vocab * p->lanes * p->v;
  if (table * 6 > EF_SMEM) return false;
  const long long room = EF_SMEM / table, threads = EF_THREADS / p->lanes;
  p->copies = (int)(room < threads ? room : threads);
  if (n < 32LL * p->copies) p->copies = (int)((n + 31) / 32);
  p->slabs = (dim + p->lanes * p->v - 1) / (p->lanes * p->v);
  if (p->slabs > 65535) return false;
  // One wave of blocks, at least 32 positions per table.
  long long blocks = sb_sm_count() / p->slabs;
  const long long most = (n + 32LL * p->copies - 1) / (32LL * p->copies);
  if (blocks > most) blocks = most;
  if (blocks < 1) blocks = 1;
  const long long per = (n + blocks * p->copies - 1) / (blocks * p->copies);
  p->per = (int)((per + 7) / 8 * 8);
  p->blocks = (int)((n + (long long)p->per * p->copies - 1) / ((long long)p->per * p->copies));
  return true;
}

struct GradPlan {
  SortPlan sort;
  int run_len, runs, group;
  size_t keys, pos, counts, totals, run_key, carry, bytes;    // byte offsets
};

GradPlan grad_plan(long long n, int vocab, int dim, int v) {
  GradPlan p;
  p.sort = sort_plan(n, vocab);
  p.group = 1;
  while (p.group < (dim + v - 1) / v && p.group < 256) p.group *= 2;
  // About two waves of runs (of 1024 threads per SM), none shorter than 32 steps.
  const long long steps = n + vocab, waves = 2LL * sb_sm_count() * (1024 / p.group);
  long long len = (steps + waves - 1) / waves;
  len = len < 32 ? 32 : len > 512 ? 512 : len;
  const long long fit = 5120 / (256 / p.group);              // the block's tokens and positions in 40 KB
  if (len > fit) len = fit;
  p.run_len = (int)len;
  p.runs = (int)((steps + len - 1) / len);
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  p.keys = take(2 * sizeof(int) * (size_t)n);                // two buffers that take turns
  p.pos = take(2 * sizeof(int) * (size_t)n);
  p.counts = take(sizeof(int) * ((size_t)1 << p.sort.bits) * (size_t)p.sort.chunks);
  p.totals = take(sizeof(int) * ((size_t)1 << p.sort.bits));
  p.run_key = take(sizeof(int) * ((size_t)p.runs + 1));
  p.carry = take(sizeof(float) * (size_t)p.runs * (size_t)dim);
  p.bytes = at;
  return p;
}

template <bool FIRST>
int launch_sort_pass(const SortArgs& a, const SortPlan& p, cudaStream_t s) {
  const int bins = 1 << p.bits;
  SB_CUDA(sb_launch(token_count_kernel<FIRST>, dim3(p.chunks), dim3(ES_THREADS), 0, s, 1, a));
  SB_COUNT_LAUNCH();
  SB_CUDA(sb_launch(token_scan_kernel, dim3((bins + 7) / 8), dim3(256), 0, s, 1, a));
  SB_COUNT_LAUNCH();
  const size_t smem = sizeof(int) * bins + sizeof(unsigned short) * bins * ES_WARPS;   // at most 40 KB
  if (p.rounds == 16) SB_CUDA(sb_launch(token_scatter_kernel<FIRST, 16>, dim3(p.chunks), dim3(ES_THREADS), smem, s, 1, a));
  else SB_CUDA(sb_launch(token_scatter_kernel<FIRST, 4>, dim3(p.chunks), dim3(ES_THREADS), smem, s, 1, a));
  SB_COUNT_LAUNCH();
  return SB_OK;
}

template <typename T, int V>
int launch_grad(GradArgs& a, cudaStream_t s) {
  const int threads = (a.dim + V - 1) / V, groups = 256 / a.group;
  const dim3 grid((a.runs + groups - 1) / groups, (threads + a.group - 1) / a.group);
  SB_CUDA(sb_launch(embedding_grad_kernel<T, V>, grid, dim3(256), 2 * sizeof(int) * (size_t)(groups * a.run_len), s, 1, a));
  SB_COUNT_LAUNCH();
  return SB_OK;
}

// Columns per thread: as dout and the fp32 table allow.
int grad_width(const void* dout, long long ld_dout, const float* dtable, long long ld_dtable, int dim, int item) {
  const int v = sb_vector_width(dout, ld_dout, dim, item, 16 / item), most = v > 4 ? 4 : v;
  const int w = sb_vector_width(dtable, ld_dtable, dim, 4, most);
  return w < most ? w : v;
}

template <typename T>
int launch_grad_type(GradArgs& a, int v, cudaStream_t s) {
  constexpr int MOST = 16 / sizeof(T);
  if (v == 8) return launch_grad<T, MOST>(a, s);
  if (v == 4) return launch_grad<T, 4>(a, s);
  if (v == 2) return launch_grad<T, 2>(a, s);
  return launch_grad<T, 1>(a, s);
}

template <typename T>
int launch_few(const FewArgs& a, const FewPlan& p, cudaStream_t s) {
  const size_t smem = sizeof(float) * (size_t)p.copies * a.vocab * p.lanes * p.v;
  static std::atomic<bool> ready[64];
  int dev = 0;
  SB_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64 || !ready[dev].load(std::memory_order_acquire)) {   // setting it twice is harmless
    SB_CUDA(cudaFuncSetAttribute(embedding_few_kernel<T, 1>, cudaFuncAttributeMaxDynamicSharedMemorySize, EF_SMEM));
    SB_CUDA(cudaFuncSetAttribute(embedding_few_kernel<T, 2>, cudaFuncAttributeMaxDynamicSharedMemorySize, EF_SMEM));
    if (dev >= 0 && dev < 64) ready[dev].store(true, std::memory_order_release);
  }
  const dim3 grid(p.blocks, p.slabs);
  const int threads = (p.copies * p.lanes + 31) / 32 * 32;
  if (p.v == 2) SB_CUDA(sb_launch(embedding_few_kernel<T, 2>, grid, dim3(threads), smem, s, 1, a));
  else SB_CUDA(sb_launch(embedding_few_kernel<T, 1>, grid, dim3(threads), smem, s, 1, a));
  SB_COUNT_LAUNCH();
  if (p.blocks > 1) {
    const long long size = (long long)a.vocab * a.dim;
    SB_CUDA(sb_launch(embedding_few_join_kernel, dim3((unsigned)((size + 31) / 32)), dim3(1024), 0, s, 1, a, p.blocks));
    SB_COUNT_LAUNCH();
  }
  return SB_OK;
}

template <typename I, typename T, typename O, int V>
cudaError_t launch_lookup(const void* tokens, const void* table, void* out, long long n, int vocab, int dim, long long ld_table,
                          long long ld_out, float scale, cudaStream_t s) {
  const long long blocks = (n * (dim / V) + 255) / 256, most = 16LL * sb_sm_count();
  return sb_launch(embedding_kernel<I, T, O, V>, dim3((unsigned)(blocks < most ? blocks : most)), dim3(256), 0, s, 1, (const I*)tokens,
                   (const T*)table, (O*)out, n, vocab, dim, ld_table, ld_out, scale);
}

template <typename I, typename T, typename O>
cudaError_t launch_lookup_width(const void* tokens, const void* table, void* out, long long n, int vocab, int dim, long long ld_table,
                                long long ld_out, float scale, cudaStream_t s) {
  constexpr int SMALL = sizeof(T) < sizeof(O) ? sizeof(T) : sizeof(O);
  constexpr int MOST = SMALL == 4 ? 4 : (sizeof(T) == sizeof(O) ? 8 : 4);
  int v = sb_vector_width(table, ld_table, dim, sizeof(T), MOST);
  v = sb_vector_width(out, ld_out, dim, sizeof(O), v);
  if (v == 8) return launch_lookup<I, T, O, MOST>(tokens, table, out, n, vocab, dim, ld_table, ld_out, scale, s);
  if (v == 4) return launch_lookup<I, T, O, 4>(tokens, table, out, n, vocab, dim, ld_table, ld_out, scale, s);
  if (v == 2) return launch_lookup<I, T, O, 2>(tokens, table, out, n, vocab, dim, ld_table, ld_out, scale, s);
  return launch_lookup<I, T, O, 1>(tokens, table, out, n, vocab, dim, ld_table, ld_out, scale, s);
}

template <typename I, typename T>
cudaError_t launch_lookup_out(int out_dtype, const void* tokens, const void* table, void* out, long long n, int vocab, int dim,
                              long long ld_table, long long ld_out, float scale, cudaStream_t s) {
  if (out_dtype == SB_F32) return launch_lookup_width<I, T, float>(tokens, table, out, n, vocab, dim, ld_table, ld_out, scale, s);
  if (out_dtype == SB_BF16) return launch_lookup_width<I, T, __nv_bfloat16>(tokens, table, out, n, vocab, dim, ld_table, ld_out, scale, s);
  return launch_lookup_width<I, T, __half>(tokens, table, out, n, vocab, dim, ld_table, ld_out, scale, s);
}

template <typename I>
cudaError_t launch_lookup_table(int table_dtype, int out_dtype, const void* tokens, const void* table, void* out, long long n, int vocab,
                                int dim, long long ld_table, long long ld_out, float scale, cudaStream_t s) {
  if (table_dtype == SB_F32) return launch_lookup_out<I, float>(out_dtype, tokens, table, out, n, vocab, dim, ld_table, ld_out, scale, s);
  if (table_dtype == SB_BF16)
    return launch_lookup_out<I, __nv_bfloat16>(out_dtype, tokens, table, out, n, vocab, dim, ld_table, ld_out, scale, s);
  return launch_lookup_out<I, __half>(out_dtype, tokens, table, out, n, vocab, dim, ld_table, ld_out, scale, s);
}

bool embed_dtype_ok(int dt) { return dt == SB_F32 || dt == SB_BF16 || dt == SB_F16; }
bool aligned_to(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

}  // namespace

extern "C" {

int sb_embedding(const void* tokens, int index_dtype, long long n, const void* table, long long ld_table, int table_dtype, int vocab, int dim,
                 float scale, void* out, long long ld_out, int out_dtype, void* stream) {
  if (n < 0 || vocab < 0 || dim < 0) return sb_fail(SB_ERR_BAD_ARG, "sb_embedding: negative size");
  if (index_dtype != SB_I32 && index_dtype != SB_I64) return sb_fail(SB_ERR_UNSUPPORTED, "sb_embedding: tokens are int32 or int64");
  if (!embed_dtype_ok(table_dtype) || !embed_dtype_ok(out_dtype))
    return sb_fail(SB_ERR_UNSUPPORTED, "sb_embedding: storage types are f32, bf16 and f16 (table %d, out %d)", table_dtype, out_dtype);
  if (n == 0 || dim == 0) return SB_OK;
  if (!tokens || !out || (!table && vocab > 0)) return sb_fail(SB_ERR_BAD_ARG, "sb_embedding: null pointer");
  if (ld_table < dim || ld_out < dim) return sb_fail(SB_ERR_BAD_ARG, "sb_embedding: a row pitch is shorter than the %d columns", dim);
  if (!aligned_to(tokens, index_dtype == SB_I64 ? 8 : 4) || !aligned_to(table, sb_dtype_size(table_dtype)) ||
      !aligned_to(out, sb_dtype_size(out_dtype)))
    return sb_fail(SB_ERR_MISALIGNED, "sb_embedding: a pointer is not aligned to its element size");
  cudaStream_t s = (cudaStream_t)stream;
  cudaError_t e = index_dtype == SB_I32
                      ? launch_lookup_table<int>(table_dtype, out_dtype, tokens, table, out, n, vocab, dim, ld_table, ld_out, scale, s)
                      : launch_lookup_table<long long>(table_dtype, out_dtype, tokens, table, out, n, vocab, dim, ld_table, ld_out, scale, s);
  SB_COUNT_LAUNCH();
  return sb_check_cuda(e, "sb_embedding");
}

int sb_embedding_grad_workspace_bytes(long long n, int vocab, int dim, size_t* bytes) {
  if (!bytes) return sb_fail(SB_ERR_BAD_ARG, "sb_embedding_grad_workspace_bytes: null output");
  if (n < 0 || vocab < 0 || dim < 0) return sb_fail(SB_ERR_BAD_ARG, "sb_embedding_grad_workspace_bytes: negative size");
  if (n > 0x40000000LL || vocab > 0x40000000) return sb_fail(SB_ERR_TOO_LARGE, "sb_embedding_grad: at most 2^30 tokens and a vocabulary of 2^30");
  // For whichever width the call's pointers and pitches allow.
  size_t most = 16;
  if (n == 0 || vocab == 0 || dim == 0) {
    *bytes = most;
    return SB_OK;
  }
  for (int v = 1; v <= 8; v *= 2) {
    const size_t need = grad_plan(n, vocab, dim, v).bytes;
    if (need > most) most = need;
    FewPlan few;
    if (v <= 2 && few_plan(n, vocab, dim, v, &few) && sizeof(float) * (size_t)few.blocks * (size_t)vocab * (size_t)dim > most)
      most = sizeof(float) * (size_t)few.blocks * (size_t)vocab * (size_t)dim;
  }
  *bytes = most;
  return SB_OK;
}

int sb_embedding_grad(const void* tokens, int index_dtype, long long n, const void* dout, long long ld_dout, int dout_dtype, float scale,
                      float* dtable, long long ld_dtable, int vocab, int dim, int accumulate, void* workspace, size_t workspace_bytes,
                      void* stream) {
  const char* who = "sb_embedding_grad";
  if (n < 0 || vocab < 0 || dim < 0) return sb_fail(SB_ERR_BAD_ARG, "%s: negative size", who);
  if (index_dtype != SB_I32 && index_dtype != SB_I64) return sb_fail(SB_ERR_UNSUPPORTED, "%s: tokens are int32 or int64", who);
  if (!embed_dtype_ok(dout_dtype)) return sb_fail(SB_ERR_UNSUPPORTED, "%s: storage types are f32, bf16 and f16 (got %d)", who, dout_dtype);
  if (vocab == 0 || dim == 0) return SB_OK;
  if (!dtable || (n > 0 && (!tokens || !dout))) return sb_fail(SB_ERR_BAD_ARG, "%s: null pointer", who);
  if (ld_dtable < dim || (n > 0 && ld_dout < dim)) return sb_fail(SB_ERR_BAD_ARG, "%s: a row pitch is shorter than the %d columns", who, dim);
  if (!aligned_to(dtable, 4) || (n > 0 && (!aligned_to(tokens, index_dtype == SB_I64 ? 8 : 4) || !aligned_to(dout, sb_dtype_size(dout_dtype)))))
    return sb_fail(SB_ERR_MISALIGNED, "%s: a pointer is not aligned to its element size", who);
  cudaStream_t s = (cudaStream_t)stream;
  if (n == 0) {
    if (!accumulate)
      SB_CUDA(cudaMemset2DAsync(dtable, sizeof(float) * (size_t)ld_dtable, 0, sizeof(float) * (size_t)dim, (size_t)vocab, s));
    return SB_OK;
  }
  size_t need = 0;
  int rc = sb_embedding_grad_workspace_bytes(n, vocab, dim, &need);
  if (rc != SB_OK) return rc;
  if (!workspace || workspace_bytes < need)
    return sb_fail(SB_ERR_BAD_ARG, "%s: needs a workspace of %zu bytes (got %zu)", who, need, workspace ? workspace_bytes : (size_t)0);
  if (!aligned_to(workspace, 16)) return sb_fail(SB_ERR_MISALIGNED, "%s: the workspace is not 16-byte aligned", who);
  const int item = sb_dtype_size(dout_dtype);
  const int v = grad_width(dout, ld_dout, dtable, ld_dtable, dim, item);
  FewPlan few;
  if (few_plan(n, vocab, dim, sb_vector_width(dout, ld_dout, dim, item, 2), &few)) {
    FewArgs f;
    memset(&f, 0, sizeof(f));
    f.tokens = tokens; f.dout = dout; f.dtable = dtable; f.partial = (float*)workspace; f.ld_dout = ld_dout; f.ld_dtable = ld_dtable;
    f.n = (int)n; f.vocab = vocab; f.dim = dim; f.index64 = index_dtype == SB_I64; f.lanes = few.lanes; f.copies = few.copies;
    f.per = few.per; f.scale = scale; f.accumulate = accumulate;
    return dout_dtype == SB_F32 ? launch_few<float>(f, few, s)
           : dout_dtype == SB_BF16 ? launch_few<__nv_bfloat16>(f, few, s) : launch_few<__half>(f, few, s);
  }
  const GradPlan p = grad_plan(n, vocab, dim, v);
  char* ws = (char*)workspace;
  SortArgs a;
  memset(&a, 0, sizeof(a));
  a.tokens = tokens; a.index64 = index_dtype == SB_I64;
  a.counts = (int*)(ws + p.counts); a.totals = (int*)(ws + p.totals);
  a.n = (int)n; a.vocab = vocab; a.bits = p.sort.bits; a.chunks = p.sort.chunks; a.chunk = p.sort.chunk;
  int* keys = (int*)(ws + p.keys);
  int* pos = (int*)(ws + p.pos);
  a.keys_out = keys; a.pos_out = pos;
  if (n <= ES_SMALL) {
    int bits = 1;
    while (bits < 31 && (1LL << bits) <= vocab) ++bits;
    const size_t smem = 6 * ES_SMALL + sizeof(unsigned short) * 256 * (ES_SMALL_THREADS / 32);   // 40 KB
    SB_CUDA(sb_launch(token_sort_small_kernel, dim3(1), dim3(ES_SMALL_THREADS), smem, s, 1, a, bits));
    SB_COUNT_LAUNCH();
  } else {
    for (int pass = 0; pass < p.sort.passes; ++pass) {
      a.shift = pass * p.sort.bits;
      a.keys_in = keys + (pass & 1 ? 0 : n); a.pos_in = pos + (pass & 1 ? 0 : n);
      a.keys_out = keys + (pass & 1 ? n : 0); a.pos_out = pos + (pass & 1 ? n : 0);
      rc = pass == 0 ? launch_sort_pass<true>(a, p.sort, s) : launch_sort_pass<false>(a, p.sort, s);
      if (rc != SB_OK) return rc;
    }
  }
  GradArgs g;
  memset(&g, 0, sizeof(g));
  g.keys = a.keys_out; g.pos = a.pos_out; g.dout = dout; g.dtable = dtable;
  g.carry = (float*)(ws + p.carry); g.run_key = (int*)(ws + p.run_key);
  g.ld_dout = ld_dout; g.ld_dtable = ld_dtable; g.n = (int)n; g.vocab = vocab; g.dim = dim;
  g.group = p.group; g.run_len = p.run_len; g.runs = p.runs; g.scale = scale; g.accumulate = accumulate;
  rc = dout_dtype == SB_F32 ? launch_grad_type<float>(g, v, s)
       : dout_dtype == SB_BF16 ? launch_grad_type<__nv_bfloat16>(g, v, s) : launch_grad_type<__half>(g, v, s);
  if (rc != SB_OK) return rc;
  if (p.runs > 1) {
    const int most = 32 * sb_sm_count();
    SB_CUDA(sb_launch(embedding_join_kernel, dim3(p.runs - 1 < most ? p.runs - 1 : most, dim > 256 ? 4 : 1), dim3(256), 0, s, 1, g));
    SB_COUNT_LAUNCH();
  }
  return SB_OK;
}

}  // extern "C"
