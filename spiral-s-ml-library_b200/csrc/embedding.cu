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

#include <limits.h>
#include <stdlib.h>

namespace {

// ------------------------------- lookup -----------------------------------------
// `lanes` threads per row (a power of two), PACKS packs of V neighbouring elements each at a time, all loads before the first
// store; the next row's token is on its way meanwhile.  65537 x 1000 from 50001 fp32 rows, 14700 of which occur, to bf16: 190 MB, 39 us back to
// back, 4.9 TB/s, bound by what an SM has on its way rather than by memory.  Where others' writes have to leave L2 meanwhile 56 us (62 with one
// pack at a time); single elements, 999 columns 67 (92 with four at a time), 177 with an index and a division for every element.
template <typename I, typename T, typename O, int V, int PACKS>
__global__ void __launch_bounds__(256)
embedding_kernel(const I* __restrict__ tokens, const T* __restrict__ table, O* __restrict__ out, long long n, int vocab, int dim,
                 long long ld_table, long long ld_out, float scale, int lanes) {
  sb_grid_dependency_wait();
  sb_grid_dependents_launch();
  const unsigned lane = threadIdx.x & (lanes - 1), stride = lanes * V;
  const long long step = (long long)gridDim.x * (blockDim.x / lanes);
  long long r = (long long)blockIdx.x * (blockDim.x / lanes) + threadIdx.x / lanes;
  long long t = r < n ? (long long)tokens[r] : 0;
  for (; r < n; r += step) {
    const bool known = t >= 0 && t < vocab;
    const T* from = table + (known ? t : 0) * ld_table;
    O* to = out + r * ld_out;
    if (r + step < n) t = (long long)tokens[r + step];
    for (unsigned c = lane * V; c < (unsigned)dim; c += PACKS * stride) {
      SbWords<sizeof(T) * V> in[PACKS] = {};
#pragma unroll
      for (int i = 0; i < PACKS; ++i) sb_load_kept(in[i], from + c + i * stride, known && c + i * stride < (unsigned)dim);
#pragma unroll
      for (int i = 0; i < PACKS; ++i) {
        float v[V];
        sb_unpack_words<T, V>(in[i], v);
#pragma unroll
        for (int k = 0; k < V; ++k) v[k] *= scale;
        if (c + i * stride < (unsigned)dim) sb_store_f32<O, V>(to + c + i * stride, v);
      }
    }
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
  p.rounds = 16;
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
  int* counts;                   // [chunks][bins], turned into the bins' running sums by the scan
  int* totals;                   // [bins]
  int n, vocab, shift, bits, chunks, chunk;
  int index64;
};

// N tokens of a thread, `stride` apart, all on their way before the first is looked at (loads and comparisons in turn follow
// one another: 4096 tokens per block took 14 us, nearly all of it 16 latencies): -1 behind the end, vocab for no token.
struct TokenWords {
  uint32_t lo, hi;
};
__device__ __forceinline__ void load_token(TokenWords& w, const void* tokens, long long i, bool index64, bool issue) {
  w.lo = w.hi = 0u;
  if (index64)
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %3, 0;\n\t@p ld.global.nc.v2.b32 {%0, %1}, [%2];\n\t}"
                 : "+r"(w.lo), "+r"(w.hi) : "l"((const char*)tokens + i * 8), "r"((uint32_t)issue));
  else
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %2, 0;\n\t@p ld.global.nc.b32 %0, [%1];\n\t}"
                 : "+r"(w.lo) : "l"((const char*)tokens + i * 4), "r"((uint32_t)issue));
}
// The token, or `none` for one outside [0, vocab).
__device__ __forceinline__ int token_of(const TokenWords& w, bool index64, int vocab, int none) {
  return w.lo < (uint32_t)vocab && (!index64 || w.hi == 0u) ? (int)w.lo : none;
}
template <int N>
__device__ __forceinline__ void load_keys(int (&key)[N], const SortArgs& a, int first, int stride, int end) {
  TokenWords w[N];
  if (a.index64) {
#pragma unroll
    for (int k = 0; k < N; ++k) load_token(w[k], a.tokens, first + k * stride, true, first + k * stride < end);
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k) load_token(w[k], a.tokens, first + k * stride, false, first + k * stride < end);
  }
#pragma unroll
  for (int k = 0; k < N; ++k) key[k] = first + k * stride < end ? token_of(w[k], a.index64 != 0, a.vocab, a.vocab) : -1;
}
// The same of an earlier pass's keys or positions (not through the read-only path: the kernel may have written them).
template <int N>
__device__ __forceinline__ void load_pairs(int (&v)[N], const int* from, int first, int stride, int end) {
#pragma unroll
  for (int k = 0; k < N; ++k) {
    v[k] = -1;
    const bool issue = first + k * stride < end;
    asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %2, 0;\n\t@q ld.global.cg.b32 %0, [%1];\n\t}"
                 : "+r"(v[k]) : "l"(from + (issue ? first + k * stride : 0)), "r"((uint32_t)issue) : "memory");
  }
}

// The lanes of a warp whose digit of `bits` bits is this one's (a lane without a token has digit 1 << bits): a vote per bit.
__device__ __forceinline__ unsigned same_digit(int digit, int bits) {
  unsigned same = 0xffffffffu;
  for (int b = 0; b <= bits; ++b) {
    const unsigned set = __ballot_sync(0xffffffffu, (digit >> b) & 1);
    same &= (digit >> b) & 1 ? set : ~set;
  }
  return same;
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
  int key[16];                   // all on their way at once
  if (FIRST) load_keys<16>(key, a, first + (int)threadIdx.x, ES_THREADS, last);
  else load_pairs<16>(key, a.keys_in, first + (int)threadIdx.x, ES_THREADS, last);
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    const int digit = key[k] < 0 ? bins : (key[k] >> a.shift) & (bins - 1);
    const unsigned same = same_digit(digit, a.bits);
    if (digit < bins && (same & ((1u << (threadIdx.x & 31)) - 1u)) == 0u) atomicAdd(&hist[digit], __popc(same));
  }
  __syncthreads();
  for (int b = threadIdx.x; b < bins; b += ES_THREADS) a.counts[(long long)blockIdx.x * bins + b] = hist[b];
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

// Running sums of the bins' counts over the chunks, and their totals: 32 neighbouring bins per block, each of its 32 warps a
// run of chunks.
__global__ void __launch_bounds__(1024) token_scan_kernel(SortArgs a) {
  __shared__ int part[32][33];
  sb_grid_dependency_wait();
  sb_grid_dependents_launch();
  const int bins = 1 << a.bits, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, bin = blockIdx.x * 32 + lane;
  const int per = (a.chunks + 31) / 32, from = min(a.chunks, warp * per), to = min(a.chunks, from + per);
  int sum = 0;
  if (bin < bins)
    for (int c = from; c < to; ++c) sum += a.counts[(long long)c * bins + bin];
  part[warp][lane] = sum;
  __syncthreads();
  int before = 0;
  for (int w = 0; w < warp; ++w) before += part[w][lane];
  if (bin >= bins) return;
  for (int c = from; c < to; ++c) {
    int* at = a.counts + (long long)c * bins + bin;
    const int here = *at;
    *at = before;
    before += here;
  }
  if (warp == 31) a.totals[bin] = before;
}

// Puts a chunk's (token, position) pairs where they belong by this digit, those of equal digits in their order: a warp
// takes a run of consecutive tokens 32 at a time; equal digits within the 32 find each other by votes.
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
  // Exclusive sums of the bins' totals: each thread a run of at most 8 bins.
  constexpr int PER = ES_MAX_BINS / ES_THREADS;
  const int per = (bins + ES_THREADS - 1) / ES_THREADS;
  int total[PER], before_me[PER], mine = 0;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int b = threadIdx.x * per + k;
    const bool in = k < per && b < bins;
    total[k] = in ? a.totals[b] : 0;
    before_me[k] = in ? a.counts[(long long)blockIdx.x * bins + b] : 0;
    mine += total[k];
  }
  const int incl = warp_inclusive(mine);
  if (lane == 31) warp_total[warp] = incl;
  __syncthreads();
  int run = incl - mine;
  for (int w = 0; w < warp; ++w) run += warp_total[w];
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int b = threadIdx.x * per + k;
    if (k < per && b < bins) base[b] = run + before_me[k];
    run += total[k];
  }
  const int first = blockIdx.x * a.chunk + warp * (32 * ROUNDS);
  int key[ROUNDS];
  unsigned short rank[ROUNDS];
  unsigned short* mine_seen = seen + warp * bins;
  if (FIRST) load_keys<ROUNDS>(key, a, first + lane, 32, a.n);
  else load_pairs<ROUNDS>(key, a.keys_in, first + lane, 32, a.n);
  int pos[ROUNDS];
  if (!FIRST) load_pairs<ROUNDS>(pos, a.pos_in, first + lane, 32, a.n);
#pragma unroll
  for (int k = 0; k < ROUNDS; ++k) {
    const int digit = key[k] < 0 ? bins : (key[k] >> a.shift) & (bins - 1);
    const unsigned same = same_digit(digit, a.bits);
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
    a.pos_out[to] = FIRST ? i : pos[k];
  }
}

// Up to ES_CLUSTER (98304) tokens in one launch: the blocks of a cluster hold the tokens in registers, at most 10 bits at a time;
// their counts meet in shared memory across the cluster, the pairs go through the workspace (L2).  The whole gradient of 64
// fp32 columns, 16384 / 65537 tokens of 50001: 27 / 37 us, 42 / 46 with two passes of three launches; 131072 of 2000 41 us, 34 with one
// such pass.  Up to ES_SMALL tokens a single block.
constexpr int ES_SMALL = 4096;
constexpr int ES_BLOCKS = 16;                                // more than the 8 that every GPU takes; B200 does
constexpr int ES_ROUNDS = 6;
constexpr int ES_CLUSTER_THREADS = 1024;
constexpr int ES_CLUSTER_BITS = 10;                          // of a digit, at most: a bin per thread
constexpr int ES_CLUSTER = ES_BLOCKS * ES_ROUNDS * ES_CLUSTER_THREADS;
constexpr int ES_SMEM = 112 * 1024;                          // at most: the pairs, and every warp's counts
__global__ void __launch_bounds__(ES_CLUSTER_THREADS) token_sort_kernel(SortArgs a, int* keys, int* pos, int bits, int rounds) {
  constexpr int WARPS = ES_CLUSTER_THREADS / 32;
  __shared__ int totals[ES_CLUSTER_THREADS], base[ES_CLUSTER_THREADS], here[ES_CLUSTER_THREADS], warp_total[2][WARPS];
  extern __shared__ int s_pairs[];                           // this block's pairs in the order of the digit
  int* s_key = s_pairs;
  int* s_pos = s_pairs + ES_CLUSTER_THREADS * rounds;
  const int bins = 1 << a.bits;                              // a thread each
  unsigned short* seen = reinterpret_cast<unsigned short*>(s_pos + ES_CLUSTER_THREADS * rounds);   // [warps][bins]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  unsigned short* mine = seen + warp * bins;
  const int rank = blockIdx.x, blocks = gridDim.x;           // the grid is one cluster
  sb_grid_dependency_wait();
  sb_grid_dependents_launch();
  const int first = (rank * ES_CLUSTER_THREADS + warp * 32) * rounds + lane;
  int key[ES_ROUNDS];
  unsigned short rank_in[ES_ROUNDS];
  int turn = 0;
  for (int shift = 0; shift < bits; shift += a.bits, turn ^= 1) {
    const int* pos_in = pos + (turn ? 0 : a.n);
    int* keys_out = keys + (turn ? a.n : 0);
    int* pos_out = pos + (turn ? a.n : 0);
    const int end = min(a.n, first - lane + 32 * rounds);
    if (shift == 0) load_keys<ES_ROUNDS>(key, a, first, 32, end);
    else load_pairs<ES_ROUNDS>(key, keys + (turn ? 0 : a.n), first, 32, end);
    for (int b = threadIdx.x; b < bins * WARPS / 2; b += ES_CLUSTER_THREADS) reinterpret_cast<int*>(seen)[b] = 0;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < ES_ROUNDS; ++k) {
      if (k >= rounds) break;
      const int digit = key[k] < 0 ? bins : (key[k] >> shift) & (bins - 1);
      const unsigned same = same_digit(digit, a.bits);
      const int before = __popc(same & ((1u << lane) - 1u));
      if (digit < bins) rank_in[k] = (unsigned short)(mine[digit] + before);
      __syncwarp();
      if (digit < bins && before == 0) mine[digit] = (unsigned short)(mine[digit] + __popc(same));
      __syncwarp();
    }
    __syncthreads();
    if ((int)threadIdx.x < bins) {
      int total = 0;
#pragma unroll 8
      for (int w = 0; w < WARPS; ++w) {
        const int c = seen[w * bins + threadIdx.x];
        seen[w * bins + threadIdx.x] = (unsigned short)total;
        total += c;
      }
      totals[threadIdx.x] = total;
    }
    __syncwarp();
    if (blocks > 1) cluster_sync_all(); else __syncthreads();
    // Where this block's tokens of each digit begin: among all (base) and among its own (here).
    int all = 0, before = 0, own = 0, incl = 0, own_incl = 0;
    if ((int)threadIdx.x < bins) {
      all = own = totals[threadIdx.x];
      if (blocks > 1) {
        int c[ES_BLOCKS];
#pragma unroll
        for (int r = 0; r < ES_BLOCKS; ++r)
          asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(c[r]) : "r"(map_to_cta(smem_u32(&totals[threadIdx.x]), (uint32_t)r)) : "memory");
        all = 0;
#pragma unroll
        for (int r = 0; r < ES_BLOCKS; ++r) {
          before += r < rank ? c[r] : 0;
          all += c[r];
        }
      }
    }
    incl = warp_inclusive(all);
    own_incl = warp_inclusive(own);
    if (lane == 31) {
      warp_total[0][warp] = incl;
      warp_total[1][warp] = own_incl;
    }
    __syncthreads();
    if ((int)threadIdx.x < bins) {
      int run = incl - all, own_run = own_incl - own;
      for (int w = 0; w < warp; ++w) {
        run += warp_total[0][w];
        own_run += warp_total[1][w];
      }
      base[threadIdx.x] = run + before - own_run;
      here[threadIdx.x] = own_run;
    }
    __syncthreads();
    int at[ES_ROUNDS];
    if (shift != 0) load_pairs<ES_ROUNDS>(at, pos_in, first, 32, end);
    // Through shared memory, so that tokens of one digit leave side by side: a scattered 4-byte store costs a clock per lane.
#pragma unroll
    for (int k = 0; k < ES_ROUNDS; ++k)
      if (key[k] >= 0) {
        const int i = first + k * 32, digit = (key[k] >> shift) & (bins - 1), to = here[digit] + mine[digit] + rank_in[k];
        s_key[to] = key[k];
        s_pos[to] = shift == 0 ? i : at[k];
      }
    __syncthreads();
    const int block_first = rank * ES_CLUSTER_THREADS * rounds, count = min(a.n - block_first, ES_CLUSTER_THREADS * rounds);
    for (int j = threadIdx.x; j < count; j += ES_CLUSTER_THREADS) {
      const int k = s_key[j], to = base[(k >> shift) & (bins - 1)] + j;
      keys_out[to] = k;
      pos_out[to] = s_pos[j];
    }
    // The pairs are where the next pass reads them, and nobody reads this block's totals any more.
    __syncwarp();
    if (blocks > 1) cluster_sync_all(); else __syncthreads();
  }
}

// ------------------------------ gradient ----------------------------------------
struct GradArgs {
  const int* keys;               // sorted tokens (vocab: none)
  const int* pos;
  const void* dout;
  float* dtable;
  float* carry;                  // [parts][dim]: what a block's part of the walk adds to the row that it leaves unfinished
  int* part_key;                 // [parts + 1]: tokens consumed where a part begins
  long long ld_dout, ld_dtable;
  int n, vocab, dim;
  int run_len;                   // steps (rows read + rows written) per run
  int parts, part_len;           // blocks, and steps of each
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
// shared memory; a group of threads per run, PACKS times V neighbouring columns per thread, the next UNROLL rows of dout on their way
// while the ones before are added.  Rows that only single elements fit have four of those per thread: 60000 x 333 of 5000 57 us,
// 88 with one; 336 columns 38.  (Every group searching the sorted tokens for itself, 17 dependent loads twice, and
// reading token and position from global memory in the loop: 50001 x 1000 fp32 213 us.)
template <typename T, int V, int PACKS>
__global__ void __launch_bounds__(256, 3) embedding_grad_kernel(GradArgs a) {
  constexpr int UNROLL = 8, W = V * PACKS;
  extern __shared__ __align__(16) int s_walk[];
  __shared__ int ends[2];
  const int groups = blockDim.x / a.group;
  const int steps = groups * a.run_len;
  float* s_carry = reinterpret_cast<float*>(s_walk);         // [256][W]: what each run leaves behind
  int* s_end = s_walk + 256 * W;                             // [groups]: the row that the run ends in
  int* s_key = s_end + groups;
  int* s_pos = s_key + steps;
  const long long first = (long long)blockIdx.x * steps, all = (long long)a.n + a.vocab;
  sb_grid_dependency_wait();
  sb_grid_dependents_launch();
  if (threadIdx.x < 64) {
    const int which = threadIdx.x >> 5;
    const int k = walk_split(a.keys, a.n, a.vocab, min(which == 0 ? first : first + steps, all));
    if ((threadIdx.x & 31) == 0) {
      ends[which] = k;
      if (blockIdx.y == 0) {                                 // of this block's part, and the next one's begin
        if (which == 0) a.part_key[blockIdx.x] = k;
        else if (blockIdx.x == gridDim.x - 1) a.part_key[gridDim.x] = k;
      }
    }
  }
  __syncthreads();
  const int k_first = ends[0], count = ends[1] - k_first;
  for (int i = threadIdx.x; i < count; i += blockDim.x) {
    s_key[i] = a.keys[k_first + i];
    s_pos[i] = a.pos[k_first + i];
  }
  __syncthreads();
  const int in_group = threadIdx.x % a.group, g = threadIdx.x / a.group;
  const int stride = a.group * V, col = blockIdx.y * PACKS * stride + in_group * V;   // of the first pack
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
  const long long d0 = min(first + (long long)g * a.run_len, all), d1 = min(d0 + a.run_len, all);
  int k = split(d0);
  const int k_end = split(d1);
  const int row0 = (int)(d0 - (k_first + k)), row_end = (int)(d1 - (k_first + k_end));
  const bool active = col < a.dim;
  bool has[PACKS];
#pragma unroll
  for (int p = 0; p < PACKS; ++p) has[p] = col + p * stride < a.dim;
  int row = row0;
  const T* dout = (const T*)a.dout + (active ? col : 0);
  float* to = a.dtable + (long long)row * a.ld_dtable + col;
  float acc[W];
#pragma unroll
  for (int t = 0; t < W; ++t) acc[t] = 0.f;
  auto finish = [&]() {
#pragma unroll
    for (int p = 0; p < PACKS; ++p) {
      float out[V];
#pragma unroll
      for (int t = 0; t < V; ++t) out[t] = acc[p * V + t] * a.scale;
      if (has[p]) {
        float* at = to + p * stride;
        if (a.accumulate) {
#pragma unroll
          for (int t = 0; t < V; ++t) out[t] += at[t];
        }
#pragma unroll
        for (int t = 0; t < V; t += 4) {
          if constexpr (V >= 4) sb_store_f32<float, 4>(at + t, out + t);
          else sb_store_f32<float, V>(at, out);
        }
      }
    }
#pragma unroll
    for (int t = 0; t < W; ++t) acc[t] = 0.f;
    to += a.ld_dtable;
    ++row;
  };
  if (active) {
    while (k < k_end) {
      SbWords<sizeof(T) * V> in[UNROLL][PACKS] = {};
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) {
        const bool issue = k + u < k_end && s_key[k + u] < a.vocab;
        const T* from = dout + (long long)(issue ? s_pos[k + u] : 0) * a.ld_dout;
#pragma unroll
        for (int p = 0; p < PACKS; ++p) sb_load_words(in[u][p], from + p * stride, issue && has[p]);
      }
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) {
        const int key = k + u < k_end ? s_key[k + u] : a.vocab;
        if (key < a.vocab) {
          while (row < key) finish();
          float v[W];
#pragma unroll
          for (int p = 0; p < PACKS; ++p) sb_unpack_words<T, V>(in[u][p], v + p * V);
#pragma unroll
          for (int t = 0; t < W; ++t) acc[t] += v[t];
        }
      }
      k += UNROLL;
    }
    while (row < row_end) finish();
  }
  // What is left belongs to the row that the next run begins in.  Where a run finishes the row that it begins in, it adds
  // what the block's runs before it left for that row, in their order; the block's last leftover goes to the workspace.
#pragma unroll
  for (int t = 0; t < W; ++t) s_carry[threadIdx.x * W + t] = acc[t];
  if (in_group == 0) s_end[g] = row_end;
  __syncthreads();
  if (!active) return;
  auto leftover = [&](int last, int r, float* sum) {         // of the runs up to `last` that end in row r
    int from = last;
    while (from > 0 && s_end[from - 1] == r) --from;
#pragma unroll
    for (int t = 0; t < W; ++t) sum[t] = 0.f;
    for (int h = from; h <= last; ++h)
#pragma unroll
      for (int t = 0; t < W; ++t) sum[t] += s_carry[(h * a.group + in_group) * W + t];
  };
  float sum[W];
  if (g > 0 && row_end > row0) {
    leftover(g - 1, row0, sum);
    float* at = a.dtable + (long long)row0 * a.ld_dtable + col;
#pragma unroll
    for (int t = 0; t < W; ++t)
      if (has[t / V]) at[t / V * stride + t % V] += sum[t] * a.scale;
  }
  if (g == groups - 1) {
    leftover(g, row_end, sum);
#pragma unroll
    for (int t = 0; t < W; ++t)
      if (has[t / V]) a.carry[(long long)blockIdx.x * a.dim + col + t / V * stride + t % V] = sum[t];
  }
}

// Few tokens in one launch: a block has neighbouring rows of the table to itself, picks the tokens that are theirs out of all,
// sorts them by counting the ones before each, and goes through its rows; nothing crosses blocks.  Bound by latency and by writing
// the table.  Against the sort, walk and join in three launches: 1 token of 2439, 369 columns 3.2 us (13.4), 256 of 5611, 37 columns
// 7.0 (15.9), 256 of 70000, 64 columns 8.5 (19.5); 256 positions of one token 28 (15.6), 128 of them 19 (19).  A call's host time
// falls from 13 to 8 us.
constexpr int GRAD_FEW_TOKENS = 256;
template <typename T, int V, int PACKS>
__global__ void __launch_bounds__(GRAD_FEW_TOKENS, 4) embedding_scan_kernel(GradArgs a, const void* tokens, int index64, int rows) {
  __shared__ __align__(16) int s_raw[GRAD_FEW_TOKENS];
  __shared__ int s_key[GRAD_FEW_TOKENS], s_pos[GRAD_FEW_TOKENS], s_count;
  const int first = blockIdx.x * rows, last = (int)min((long long)first + rows, (long long)a.vocab);
  if (threadIdx.x == 0) s_count = 0;
  __syncthreads();
  sb_grid_dependency_wait();
  sb_grid_dependents_launch();
  long long token = -1;
  if ((int)threadIdx.x < a.n) token = index64 ? ((const long long*)tokens)[threadIdx.x] : (long long)((const int*)tokens)[threadIdx.x];
  const bool mine = token >= first && token < last;
  s_raw[threadIdx.x] = mine ? (int)token : INT_MAX;          // last in the order, and no key is as large
  const unsigned with = __ballot_sync(0xffffffffu, mine);
  if ((threadIdx.x & 31) == 0 && with) atomicAdd(&s_count, __popc(with));
  __syncthreads();
  const int count = s_count;
  if (mine) {
    int before = 0;
#pragma unroll 4
    for (int i = 0; i < a.n; i += 4) {
      const int4 w = *reinterpret_cast<const int4*>(&s_raw[i]);
      const int t = (int)token, at = (int)threadIdx.x - i;   // equal ones count where they come first
      before += (w.x < t + (at > 0)) + (w.y < t + (at > 1)) + (w.z < t + (at > 2)) + (w.w < t + (at > 3));
    }
    s_key[before] = (int)token;
    s_pos[before] = threadIdx.x;
  }
  __syncthreads();
  const int in_group = threadIdx.x % a.group, g = threadIdx.x / a.group, groups = blockDim.x / a.group;
  const int col = blockIdx.y * PACKS * a.group * V + in_group * V;
  const int each = (last - first + groups - 1) / groups, row0 = min(first + g * each, last), row_end = min(row0 + each, last);
  if (col >= a.dim || row0 >= row_end) return;
  auto lower = [&](int row) {                                // the first entry of `row` or behind
    int lo = 0, hi = count;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (s_key[mid] < row) lo = mid + 1;
      else hi = mid;
    }
    return lo;
  };
  // A row at a time; few have any token.
  constexpr int UNROLL = 8;
  const int stride = a.group * V;
  const T* dout = (const T*)a.dout + col;
  float* to = a.dtable + (long long)row0 * a.ld_dtable + col;
  int k = lower(row0);
  int next = k < count ? s_key[k] : INT_MAX;
  for (int row = row0; row < row_end; ++row, to += a.ld_dtable) {
    float acc[PACKS * V];
#pragma unroll
    for (int t = 0; t < PACKS * V; ++t) acc[t] = 0.f;
    if (next == row) {
      int end = k + 1;
      while (end < count && s_key[end] == row) ++end;
      for (; k < end; k += UNROLL) {
        SbWords<sizeof(T) * V> in[UNROLL][PACKS] = {};       // zeros where there is no row
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
          const bool issue = k + u < end;
          const T* from = dout + (long long)(issue ? s_pos[k + u] : 0) * a.ld_dout;
#pragma unroll
          for (int p = 0; p < PACKS; ++p) sb_load_words(in[u][p], from + p * stride, issue && col + p * stride < a.dim);
        }
#pragma unroll
        for (int u = 0; u < UNROLL; ++u)
#pragma unroll
          for (int p = 0; p < PACKS; ++p) {
            float v[V];
            sb_unpack_words<T, V>(in[u][p], v);
#pragma unroll
            for (int t = 0; t < V; ++t) acc[p * V + t] += v[t];
          }
      }
      k = end;
      next = k < count ? s_key[k] : INT_MAX;
    }
#pragma unroll
    for (int p = 0; p < PACKS; ++p) {
      if (col + p * stride >= a.dim) continue;
      float* at = to + p * stride;
#pragma unroll
      for (int t = 0; t < V; ++t) acc[p * V + t] = a.accumulate ? at[t] + acc[p * V + t] * a.scale : acc[p * V + t] * a.scale;
#pragma unroll
      for (int t = 0; t < V; t += 4) {
        if constexpr (V >= 4) sb_store_f32<float, 4>(at + t, acc + p * V + t);
        else sb_store_f32<float, V>(at, acc + p * V);
      }
    }
  }
}

// A table of few rows needs no sort: every warp (or part of one) adds its share of the positions, in their order, to a table of
// its own in shared memory, one or two columns per thread; the block adds its tables up, and the blocks' sums are
// added in their order by a second launch.  524288 x 64 bf16 over 53 tokens
// 28 us (floor 11): bound by the tables' turns of load, add and store in shared memory.
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

template <typename T, int V, int PACKS>
__global__ void __launch_bounds__(EF_THREADS) embedding_few_kernel(FewArgs a) {
  constexpr int UNROLL = 16;                                 // at most `lanes`: as many tokens as one load of the group brings
  extern __shared__ __align__(16) float s_tables[];          // [copies][vocab + 1][lanes * V * PACKS]; the last row is for no token
  const int stride = a.lanes * V, width = stride * PACKS, table = (a.vocab + 1) * width;
  const int copy = threadIdx.x / a.lanes, lane = threadIdx.x % a.lanes;
  for (int i = threadIdx.x; i < a.copies * table / 4; i += EF_THREADS) reinterpret_cast<float4*>(s_tables)[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  sb_grid_dependency_wait();
  sb_grid_dependents_launch();
  __syncthreads();
  const int col = blockIdx.y * width + lane * V;             // of the first pack
  const long long first = ((long long)blockIdx.x * a.copies + copy) * a.per;
  const int count = (int)max(0LL, min((long long)a.per, a.n - first));
  // Rows do not wait for their tokens, and the next UNROLL of both are on their way while these are added.
  float* mine = s_tables + copy * table + lane * V;
  const bool active = col < a.dim;
  const T* dout = (const T*)a.dout + (active ? first * a.ld_dout + col : 0);
  struct Ahead {
    SbWords<sizeof(T) * V> row[UNROLL][PACKS];
    TokenWords token;            // lane u holds row u's, as it was read: looking at it would wait for it
  };
  auto fetch = [&](Ahead& x, int i) {
    load_token(x.token, a.tokens, first + i + lane, a.index64 != 0, lane < UNROLL && i + lane < count);
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
#pragma unroll
      for (int p = 0; p < PACKS; ++p) {
        const bool in = col + p * stride < a.dim;
        sb_load_words(x.row[u][p], dout + (in ? (long long)(i + u) * a.ld_dout + p * stride : 0), in && i + u < count);
      }
  };
  auto add = [&](const Ahead& x, int i) {
    const int token = i + lane < count ? token_of(x.token, a.index64 != 0, a.vocab, a.vocab) : a.vocab;
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      float* to = mine + __shfl_sync(0xffffffffu, token, u, a.lanes) * width;
#pragma unroll
      for (int p = 0; p < PACKS; ++p) {
        float v[V], t[V];
        sb_unpack_words<T, V>(x.row[u][p], v);
        sb_unpack<float, V>(sb_load_pack<float, V>(to + p * stride), t);
#pragma unroll
        for (int k = 0; k < V; ++k) t[k] += v[k];
        sb_store_f32<float, V>(to + p * stride, t);
      }
    }
  };
  if (copy < a.copies) {         // whole warps; the others help before and after
    Ahead x = {}, y = {};        // by turns: a copy from one to the other would wait for the loads
    fetch(x, 0);
    for (int i = 0; i < a.per; i += 2 * UNROLL) {            // the same for all
      fetch(y, i + UNROLL);
      add(x, i);
      fetch(x, i + 2 * UNROLL);
      add(y, i + UNROLL);
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < a.vocab * width; i += EF_THREADS) {
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

// Adds what parts of the walk left unfinished to the row that a later part finished.  A warp looks at a part each; where few
// parts lead up to it, as with all but the commonest tokens, it adds them itself, and the block's warps share the others: every
// warp a run of the parts, in order, and their sums meet in shared memory.
template <int V>
__device__ __forceinline__ void join_add(float* s, const float* from) {
  float v[V];
  sb_unpack<float, V>(sb_load_pack<float, V>(from), v);
#pragma unroll
  for (int t = 0; t < V; ++t) s[t] += v[t];
}
template <int V>
__global__ void __launch_bounds__(256) embedding_join_kernel(GradArgs a) {
  constexpr int FEW = 8;
  __shared__ float sums[8][32 * V];
  __shared__ int shared_from[8], shared_to[8], shared_row[8];
  sb_grid_dependency_wait();
  sb_grid_dependents_launch();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long all = (long long)a.n + a.vocab;
  const int part = blockIdx.x * 8 + warp + 1;
  int from = part, row = 0;      // parts from .. part - 1 lead up to it
  if (part < a.parts) {
    const long long d0 = (long long)part * a.part_len, d1 = min(d0 + a.part_len, all);
    const int k0 = a.part_key[part], row_end = (int)(d1 - a.part_key[part + 1]);
    const int row_before = (int)((long long)(part - 1) * a.part_len - a.part_key[part - 1]);
    row = (int)(d0 - k0);
    // Only where this part finishes a row that tokens of earlier parts have been added to.
    if (row < a.vocab && row_end > row && k0 > 0 && a.keys[k0 - 1] == row) {
      from = part - 1;
      if (row_before == row) {   // the part before begins in the same row: look for the first that ends in it
        int lo = 0, hi = part - 1;
        while (lo < hi) {
          const int mid = (lo + hi) >> 1;
          if ((long long)(mid + 1) * a.part_len - a.part_key[mid + 1] >= row) hi = mid;
          else lo = mid + 1;
        }
        from = lo;
      }
    }
  }
  const bool many = part - from > FEW;
  if (lane == 0) {
    shared_from[warp] = many ? from : part;
    shared_to[warp] = part;
    shared_row[warp] = row;
  }
  if (!many && from < part)
    for (int c = (blockIdx.y * 32 + lane) * V; c < a.dim; c += 32 * V * gridDim.y) {
      float s[V] = {};
      for (int r = from; r < part; ++r) join_add<V>(s, a.carry + (long long)r * a.dim + c);
      float* to = a.dtable + (long long)row * a.ld_dtable + c;
#pragma unroll
      for (int t = 0; t < V; ++t) to[t] += s[t] * a.scale;
    }
  __syncthreads();
  for (int w = 0; w < 8; ++w) {
    const int begin = shared_from[w], end = shared_to[w], share = (end - begin + 7) / 8;
    if (begin >= end) continue;
    const int mine = begin + warp * share, last = min(end, mine + share);
    for (int c0 = blockIdx.y * 32 * V; c0 < a.dim; c0 += 32 * V * gridDim.y) {
      const int c = c0 + lane * V;
      float s[V] = {};
      if (c < a.dim) {
#pragma unroll 4
        for (int r = mine; r < last; ++r) join_add<V>(s, a.carry + (long long)r * a.dim + c);
      }
#pragma unroll
      for (int t = 0; t < V; ++t) sums[warp][lane * V + t] = s[t];
      __syncthreads();
      for (int i = threadIdx.x; i < 32 * V; i += 256)
        if (c0 + i < a.dim) {
          float total = 0.f;
#pragma unroll
          for (int v = 0; v < 8; ++v) total += sums[v][i];
          a.dtable[(long long)shared_row[w] * a.ld_dtable + c0 + i] += total * a.scale;
        }
      __syncthreads();
    }
  }
}

struct FewPlan {
  int v, lanes, copies, per, blocks, slabs;
};

// Copies of 64 columns of the table (two per thread, neighbours where dout allows pairs; 32 or 16, one per thread, of shorter
// rows) in a block's shared memory: nine or more of them, up to 85 rows or so.  524288 tokens, 64 columns bf16, 53 / 120 rows: 28 /
// 56 us (14 / 6 copies), sorted 42.  24116 x 1347 f16 of 16: 42 us with pairs 32 columns apart, 73 with one column per thread.
bool few_plan(long long n, int vocab, int dim, FewPlan* p) {
  p->v = dim >= 64 ? 2 : 1;
  p->lanes = 32;
  if (p->v == 1)
    while (p->lanes > 16 && p->lanes / 2 >= dim) p->lanes /= 2;
  const long long table = 4LL * (vocab + 1LL) * p->lanes * p->v;
  if (table * 9 > EF_SMEM) return false;
  const long long room = EF_SMEM / table, threads = EF_THREADS / p->lanes;
  p->copies = (int)(room < threads ? room : threads);
  if (n < 32LL * p->copies) p->copies = (int)((n + 31) / 32);
  if (p->lanes < 32) p->copies = p->copies < 2 ? 2 : p->copies / 2 * 2;        // whole warps
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
  int run_len, parts, part_len, group;
  size_t keys, pos, counts, totals, part_key, carry, bytes;   // byte offsets
};

GradPlan grad_plan(long long n, int vocab, int dim, int w) {   // w columns per thread
  GradPlan p;
  p.sort = sort_plan(n, vocab);
  p.group = 1;
  while (p.group < (dim + w - 1) / w && p.group < 256) p.group *= 2;
  // Runs of 8 to 512 steps: one wave of 768 threads per SM, whose blocks share the search for their part; two and a half where a
  // run has most of a block (524288 tokens of 2000, 64 columns 50 us against 63; 65537 of 50001, 1000 columns 132 against 123).
  const long long steps = n + vocab, waves = (long long)sb_sm_count() * (p.group >= 128 ? 2048 : 768) / p.group;
  long long len = (steps + waves - 1) / waves;
  len = len < 8 ? 8 : len > 512 ? 512 : len;
  const long long fit = 4096 / (256 / p.group);              // the block's tokens and positions in 32 KB
  if (len > fit) len = fit;
  p.run_len = (int)len;
  p.part_len = (int)(len * (256 / p.group));
  p.parts = (int)((steps + p.part_len - 1) / p.part_len);
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
  p.part_key = take(sizeof(int) * ((size_t)p.parts + 1));
  p.carry = take(sizeof(float) * (size_t)p.parts * (size_t)dim);
  p.bytes = at;
  return p;
}

template <bool FIRST>
int launch_sort_pass(const SortArgs& a, const SortPlan& p, cudaStream_t s) {
  const int bins = 1 << p.bits;
  SB_CUDA(sb_launch(token_count_kernel<FIRST>, dim3(p.chunks), dim3(ES_THREADS), 0, s, 1, a));
  SB_COUNT_LAUNCH();
  SB_CUDA(sb_launch(token_scan_kernel, dim3((bins + 31) / 32), dim3(1024), 0, s, 1, a));
  SB_COUNT_LAUNCH();
  const size_t smem = sizeof(int) * bins + sizeof(unsigned short) * bins * ES_WARPS;   // at most 40 KB
  SB_CUDA(sb_launch(token_scatter_kernel<FIRST, 16>, dim3(p.chunks), dim3(ES_THREADS), smem, s, 1, a));
  SB_COUNT_LAUNCH();
  return SB_OK;
}

template <typename T, int V, int PACKS>
int launch_grad(GradArgs& a, cudaStream_t s) {
  const int threads = (a.dim + V * PACKS - 1) / (V * PACKS), groups = 256 / a.group;
  const dim3 grid(a.parts, (threads + a.group - 1) / a.group);
  const size_t smem = sizeof(int) * (size_t)(256 * V * PACKS + groups + 2 * a.part_len);   // at most 41 KB
  SB_CUDA(sb_launch(embedding_grad_kernel<T, V, PACKS>, grid, dim3(256), smem, s, 1, a));
  SB_COUNT_LAUNCH();
  return SB_OK;
}

// Columns per thread: as dout and the fp32 table allow.
int grad_width(const void* dout, long long ld_dout, const float* dtable, long long ld_dtable, int dim, int item) {
  const int v = sb_vector_width(dout, ld_dout, dim, item, 16 / item), most = v > 4 ? 4 : v;
  const int w = sb_vector_width(dtable, ld_dtable, dim, 4, most);
  return w < most ? w : v;
}

template <typename T, int V, int PACKS>
int launch_scan(GradArgs& a, const void* tokens, int index64, cudaStream_t s) {
  a.group = 1;
  while (a.group < (a.dim + V * PACKS - 1) / (V * PACKS) && a.group < 256) a.group *= 2;
  // Sixteen blocks per SM (200 tokens of 50001, 1000 columns 37 us, 54 with four), or a row per group.
  const int groups = GRAD_FEW_TOKENS / a.group, most = 16 * sb_sm_count();
  const int threads = (a.dim + V * PACKS - 1) / (V * PACKS), slabs = (threads + a.group - 1) / a.group;
  int rows = (int)(((long long)a.vocab * slabs + most - 1) / most);
  if (rows < groups) rows = groups;
  SB_CUDA(sb_launch(embedding_scan_kernel<T, V, PACKS>, dim3((unsigned)((a.vocab + (long long)rows - 1) / rows), slabs), dim3(GRAD_FEW_TOKENS), 0, s, 1, a,
                    tokens, index64, rows));
  SB_COUNT_LAUNCH();
  return SB_OK;
}

template <typename T>
int launch_scan_type(GradArgs& a, int v, const void* tokens, int index64, cudaStream_t s) {
  constexpr int MOST = 16 / sizeof(T);
  if (v == 8) return launch_scan<T, MOST, 1>(a, tokens, index64, s);
  if (v == 4) return launch_scan<T, 4, 1>(a, tokens, index64, s);
  if (v == 2) return launch_scan<T, 2, 2>(a, tokens, index64, s);
  return launch_scan<T, 1, 4>(a, tokens, index64, s);
}

template <typename T>
int launch_grad_type(GradArgs& a, int v, cudaStream_t s) {
  constexpr int MOST = 16 / sizeof(T);
  if (v == 8) return launch_grad<T, MOST, 1>(a, s);
  if (v == 4) return launch_grad<T, 4, 1>(a, s);
  if (v == 2) return launch_grad<T, 2, 2>(a, s);
  return launch_grad<T, 1, 4>(a, s);
}

template <typename T>
int launch_few(const FewArgs& a, const FewPlan& p, bool pairs, cudaStream_t s) {
  const size_t smem = sizeof(float) * (size_t)p.copies * (size_t)(a.vocab + 1) * p.lanes * p.v;
  static std::atomic<bool> ready[64];
  int dev = 0;
  SB_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64 || !ready[dev].load(std::memory_order_acquire)) {   // setting it twice is harmless
    SB_CUDA(cudaFuncSetAttribute(embedding_few_kernel<T, 1, 1>, cudaFuncAttributeMaxDynamicSharedMemorySize, EF_SMEM));
    SB_CUDA(cudaFuncSetAttribute(embedding_few_kernel<T, 1, 2>, cudaFuncAttributeMaxDynamicSharedMemorySize, EF_SMEM));
    SB_CUDA(cudaFuncSetAttribute(embedding_few_kernel<T, 2, 1>, cudaFuncAttributeMaxDynamicSharedMemorySize, EF_SMEM));
    if (dev >= 0 && dev < 64) ready[dev].store(true, std::memory_order_release);
  }
  const dim3 grid(p.blocks, p.slabs);
  if (p.v == 1) SB_CUDA(sb_launch(embedding_few_kernel<T, 1, 1>, grid, dim3(EF_THREADS), smem, s, 1, a));
  else if (pairs) SB_CUDA(sb_launch(embedding_few_kernel<T, 2, 1>, grid, dim3(EF_THREADS), smem, s, 1, a));
  else SB_CUDA(sb_launch(embedding_few_kernel<T, 1, 2>, grid, dim3(EF_THREADS), smem, s, 1, a));
  SB_COUNT_LAUNCH();
  if (p.blocks > 1) {
    const long long size = (long long)a.vocab * a.dim;
    SB_CUDA(sb_launch(embedding_few_join_kernel, dim3((unsigned)((size + 31) / 32)), dim3(1024), 0, s, 1, a, p.blocks));
    SB_COUNT_LAUNCH();
  }
  return SB_OK;
}

template <typename I, typename T, typename O, int V, int PACKS>
cudaError_t launch_lookup(const void* tokens, const void* table, void* out, long long n, int vocab, int dim, long long ld_table,
                          long long ld_out, float scale, cudaStream_t s) {
  const int packs = (dim + V * PACKS - 1) / (V * PACKS);
  int lanes = 1;
  while (lanes < packs && lanes < 256) lanes *= 2;
  const long long blocks = (n * lanes + 255) / 256, most = 16LL * sb_sm_count();
  return sb_launch(embedding_kernel<I, T, O, V, PACKS>, dim3((unsigned)(blocks < most ? blocks : most)), dim3(256), 0, s, 1, (const I*)tokens,
                   (const T*)table, (O*)out, n, vocab, dim, ld_table, ld_out, scale, lanes);
}

template <typename I, typename T, typename O>
cudaError_t launch_lookup_width(const void* tokens, const void* table, void* out, long long n, int vocab, int dim, long long ld_table,
                                long long ld_out, float scale, cudaStream_t s) {
  constexpr int SMALL = sizeof(T) < sizeof(O) ? sizeof(T) : sizeof(O);
  constexpr int MOST = SMALL == 4 ? 4 : (sizeof(T) == sizeof(O) ? 8 : 4);
  int v = sb_vector_width(table, ld_table, dim, sizeof(T), MOST);
  v = sb_vector_width(out, ld_out, dim, sizeof(O), v);
  if (v == 8) return launch_lookup<I, T, O, MOST, 2>(tokens, table, out, n, vocab, dim, ld_table, ld_out, scale, s);
  if (v == 4) return launch_lookup<I, T, O, 4, 2>(tokens, table, out, n, vocab, dim, ld_table, ld_out, scale, s);
  if (v == 2) return launch_lookup<I, T, O, 2, 4>(tokens, table, out, n, vocab, dim, ld_table, ld_out, scale, s);
  return launch_lookup<I, T, O, 1, 8>(tokens, table, out, n, vocab, dim, ld_table, ld_out, scale, s);
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

// Whether n tokens are sorted in one launch: by one block, or by a cluster of ES_BLOCKS where the device has room for one, which
// it is asked once (a part of it, or one with fewer SMs side by side, need not have).  SB_SORT_CLUSTER=0 in the environment: never a cluster.
int token_sort_fits(long long n, bool* fits) {
  static std::atomic<int> known[64];                         // 1: one block only, 2: a cluster too
  int dev = 0;
  SB_CUDA(cudaGetDevice(&dev));
  const bool keep = dev >= 0 && dev < 64;
  int state = keep ? known[dev].load(std::memory_order_acquire) : 0;
  if (state == 0) {                                          // asking twice is harmless
    SB_CUDA(cudaFuncSetAttribute(token_sort_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, ES_SMEM));
    state = 1;
    const char* e = getenv("SB_SORT_CLUSTER");
    if (!(e && e[0] == '0') && cudaFuncSetAttribute(token_sort_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess) {
      cudaLaunchConfig_t cfg;
      memset(&cfg, 0, sizeof(cfg));
      cfg.gridDim = dim3(ES_BLOCKS);
      cfg.blockDim = dim3(ES_CLUSTER_THREADS);
      cfg.dynamicSmemBytes = ES_SMEM;
      cudaLaunchAttribute attr;
      attr.id = cudaLaunchAttributeClusterDimension;
      attr.val.clusterDim.x = ES_BLOCKS;
      attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
      cfg.attrs = &attr;
      cfg.numAttrs = 1;
      int clusters = 0;
      if (cudaOccupancyMaxActiveClusters(&clusters, token_sort_kernel, &cfg) == cudaSuccess && clusters > 0) state = 2;
    }
    if (state == 1) cudaGetLastError();                      // an answer of "no" is none of the caller's errors
    if (keep) known[dev].store(state, std::memory_order_release);
  }
  *fits = n <= ES_SMALL || (n <= ES_CLUSTER && state == 2);
  return SB_OK;
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
  // For whichever number of columns per thread the call's pointers and pitches allow.
  size_t most = 16;
  if (n == 0 || vocab == 0 || dim == 0) {
    *bytes = most;
    return SB_OK;
  }
  FewPlan few;
  if (few_plan(n, vocab, dim, &few)) {
    const size_t need = sizeof(float) * (size_t)few.blocks * (size_t)vocab * (size_t)dim;
    if (need > most) most = need;
  } else {
    for (int w = 4; w <= 8; w *= 2) {
      const size_t need = grad_plan(n, vocab, dim, w).bytes;
      if (need > most) most = need;
    }
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
  if (few_plan(n, vocab, dim, &few)) {
    FewArgs f;
    memset(&f, 0, sizeof(f));
    f.tokens = tokens; f.dout = dout; f.dtable = dtable; f.partial = (float*)workspace; f.ld_dout = ld_dout; f.ld_dtable = ld_dtable;
    f.n = (int)n; f.vocab = vocab; f.dim = dim; f.index64 = index_dtype == SB_I64; f.lanes = few.lanes; f.copies = few.copies;
    f.per = few.per; f.scale = scale; f.accumulate = accumulate;
    const bool pairs = sb_vector_width(dout, ld_dout, dim, item, 2) == 2;
    return dout_dtype == SB_F32 ? launch_few<float>(f, few, pairs, s)
           : dout_dtype == SB_BF16 ? launch_few<__nv_bfloat16>(f, few, pairs, s) : launch_few<__half>(f, few, pairs, s);
  }
  if (n <= GRAD_FEW_TOKENS) {
    GradArgs g;
    memset(&g, 0, sizeof(g));
    g.dout = dout; g.dtable = dtable; g.ld_dout = ld_dout; g.ld_dtable = ld_dtable; g.n = (int)n; g.vocab = vocab; g.dim = dim;
    g.scale = scale; g.accumulate = accumulate;
    const int index64 = index_dtype == SB_I64;
    return dout_dtype == SB_F32 ? launch_scan_type<float>(g, v, tokens, index64, s)
           : dout_dtype == SB_BF16 ? launch_scan_type<__nv_bfloat16>(g, v, tokens, index64, s) : launch_scan_type<__half>(g, v, tokens, index64, s);
  }
  const GradPlan p = grad_plan(n, vocab, dim, v < 4 ? 4 : v);
  char* ws = (char*)workspace;
  SortArgs a;
  memset(&a, 0, sizeof(a));
  a.tokens = tokens; a.index64 = index_dtype == SB_I64;
  a.counts = (int*)(ws + p.counts); a.totals = (int*)(ws + p.totals);
  a.n = (int)n; a.vocab = vocab; a.bits = p.sort.bits; a.chunks = p.sort.chunks; a.chunk = p.sort.chunk;
  int* keys = (int*)(ws + p.keys);
  int* pos = (int*)(ws + p.pos);
  a.keys_out = keys; a.pos_out = pos;
  bool one_launch = false;
  if ((rc = token_sort_fits(n, &one_launch)) != SB_OK) return rc;
  if (one_launch) {
    int bits = 1;
    while (bits < 31 && (1LL << bits) <= vocab) ++bits;
    const int passes = (bits + ES_CLUSTER_BITS - 1) / ES_CLUSTER_BITS;
    a.bits = (bits + passes - 1) / passes;
    const int blocks = n <= ES_SMALL ? 1 : ES_BLOCKS;
    const int rounds = (int)((n + (long long)blocks * ES_CLUSTER_THREADS - 1) / ((long long)blocks * ES_CLUSTER_THREADS));
    const size_t smem = 2 * sizeof(int) * (size_t)(ES_CLUSTER_THREADS * rounds) + (sizeof(short) * ES_CLUSTER_THREADS / 32 << a.bits);
    SB_CUDA(sb_launch(token_sort_kernel, dim3(blocks), dim3(ES_CLUSTER_THREADS), smem, s, blocks, a, keys, pos, bits, rounds));
    SB_COUNT_LAUNCH();
    a.keys_out = keys + (passes & 1 ? 0 : n);
    a.pos_out = pos + (passes & 1 ? 0 : n);
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
  g.carry = (float*)(ws + p.carry); g.part_key = (int*)(ws + p.part_key);
  g.ld_dout = ld_dout; g.ld_dtable = ld_dtable; g.n = (int)n; g.vocab = vocab; g.dim = dim;
  g.group = p.group; g.run_len = p.run_len; g.parts = p.parts; g.part_len = p.part_len; g.scale = scale; g.accumulate = accumulate;
  rc = dout_dtype == SB_F32 ? launch_grad_type<float>(g, v, s)
       : dout_dtype == SB_BF16 ? launch_grad_type<__nv_bfloat16>(g, v, s) : launch_grad_type<__half>(g, v, s);
  if (rc != SB_OK) return rc;
  if (p.parts > 1) {
    const int wide = v >= 4 ? 128 : 32, slabs = (dim + wide - 1) / wide;   // columns of a warp
    const dim3 grid((p.parts + 6) / 8, slabs < 8 ? slabs : 8);
    if (v >= 4) SB_CUDA(sb_launch(embedding_join_kernel<4>, grid, dim3(256), 0, s, 1, g));
    else SB_CUDA(sb_launch(embedding_join_kernel<1>, grid, dim3(256), 0, s, 1, g));
    SB_COUNT_LAUNCH();
  }
  return SB_OK;
}

}  // extern "C"
