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
  const int first = blockIdx.x * a.chunk, last = min(a.n - first, a.chunk) + first;
  for (int i = first + threadIdx.x; i < last; i += ES_THREADS)
    atomicAdd(&hist[(sort_key<FIRST>(a, i) >> a.shift) & (bins - 1)], 1);
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
// row is finished when all tokens up to it have been added.
__device__ __forceinline__ int walk_split(const int* __restrict__ keys, int n, int vocab, long long d) {
  long long lo = d > vocab ? d - vocab : 0, hi = d < n ? d : n;
  while (lo < hi) {
    const long long mid = (lo + hi) >> 1;
    if ((long long)keys[mid] <= d - 1 - mid) lo = mid + 1;
    else hi = mid;
  }
  return (int)lo;
}

// A group of threads per run, V neighbouring columns per thread; the next UNROLL rows of dout are on their way while
// the ones before are added.
template <typename T, int V>
__global__ void __launch_bounds__(256) embedding_grad_kernel(GradArgs a) {
  constexpr int UNROLL = 8;
  sb_grid_dependency_wait();
  sb_grid_dependents_launch();
  const int groups = blockDim.x / a.group;
  const int in_group = threadIdx.x % a.group;
  const int run = blockIdx.x * groups + threadIdx.x / a.group;
  const int col = (blockIdx.y * a.group + in_group) * V;
  if (run >= a.runs) return;
  const long long d0 = (long long)run * a.run_len, all = (long long)a.n + a.vocab;
  const long long d1 = d0 + a.run_len < all ? d0 + a.run_len : all;
  int k = walk_split(a.keys, a.n, a.vocab, d0);
  const int k_end = walk_split(a.keys, a.n, a.vocab, d1);
  if (blockIdx.y == 0 && in_group == 0) {
    a.run_key[run] = k;
    if (run == a.runs - 1) a.run_key[a.runs] = k_end;
  }
  if (col >= a.dim) return;
  int row = (int)(d0 - k);
  const int row_end = (int)(d1 - k_end);
  const T* dout = (const T*)a.dout + col;
  float acc[V];
#pragma unroll
  for (int t = 0; t < V; ++t) acc[t] = 0.f;
  auto finish = [&](int r) {
    float* to = a.dtable + (long long)r * a.ld_dtable + col;
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
  };
  while (k < k_end) {
    SbPack<T, V> in[UNROLL];
    int key[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      key[u] = k + u < k_end ? a.keys[k + u] : -1;
      if (key[u] >= 0 && key[u] < a.vocab) in[u] = sb_load_pack<T, V>(dout + (long long)a.pos[k + u] * a.ld_dout);
      else in[u] = sb_zero_pack<T, V>();
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      if (key[u] >= 0 && key[u] < a.vocab) {
        while (row < key[u]) finish(row++);
        float v[V];
        sb_unpack<T, V>(in[u], v);
#pragma unroll
        for (int t = 0; t < V; ++t) acc[t] += v[t];
      }
    }
    k += UNROLL;
  }
  while (row < row_end) finish(row++);
  float* carry = a.carry + (long long)run * a.dim + col;
#pragma unroll
  for (int t = 0; t < V; ++t) carry[t] = acc[t];
}

// Adds what runs left unfinished: the run that finished the row begins at, a block of 8 warps per (run, 32 columns); every
// warp takes a part of the runs before it, in order, and the warps' sums meet in shared memory.
__global__ void __launch_bounds__(256) embedding_join_kernel(GradArgs a) {
  __shared__ float sums[8][32];
  sb_grid_dependency_wait();
  sb_grid_dependents_launch();
  const int run = blockIdx.x + 1, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long d0 = (long long)run * a.run_len;
  const int k0 = a.run_key[run], row = (int)(d0 - k0);
  const long long all = (long long)a.n + a.vocab;
  const long long d1 = d0 + a.run_len < all ? d0 + a.run_len : all;
  const int row_end = (int)(d1 - a.run_key[run + 1]);
  // Only where this run finishes a row that tokens of earlier runs have been added to.
  if (row >= a.vocab || row_end == row || k0 == 0 || a.keys[k0 - 1] != row) return;
  int lo = 0, hi = run;          // the first run that begins in this row or ends in it
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if ((int)((long long)(mid + 1) * a.run_len - a.run_key[mid + 1]) >= row) hi = mid;
    else lo = mid + 1;
  }
  const int parts = run - lo, per = (parts + 7) / 8;
  const int from = lo + warp * per, to = min(run, from + per);
  for (int c = lane; c < (a.dim + 31) / 32 * 32; c += 32) {
    float s = 0.f;
    if (c < a.dim)
      for (int r = from; r < to; ++r) s += a.carry[(long long)r * a.dim + c];
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

struct GradPlan {
  SortPlan sort;
  int run_len, runs;
  size_t keys, pos, counts, totals, run_key, carry, bytes;    // byte offsets
};

GradPlan grad_plan(long long n, int vocab, int dim) {
  GradPlan p;
  p.sort = sort_plan(n, vocab);
  const long long steps = n + vocab;
  const long long least = (steps + 8191) / 8192;             // at most 8192 runs
  p.run_len = (int)(least > 32 ? least : 32);
  p.runs = (int)((steps + p.run_len - 1) / p.run_len);
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
  const int threads = (a.dim + V - 1) / V;
  int group = 1;
  while (group < threads && group < 256) group *= 2;
  a.group = group;
  const int groups = 256 / group;
  const dim3 grid((a.runs + groups - 1) / groups, (threads + group - 1) / group);
  SB_CUDA(sb_launch(embedding_grad_kernel<T, V>, grid, dim3(256), 0, s, 1, a));
  SB_COUNT_LAUNCH();
  return SB_OK;
}

template <typename T>
int launch_grad_type(GradArgs& a, cudaStream_t s) {
  constexpr int MOST = 16 / sizeof(T);
  int v = sb_vector_width(a.dout, a.ld_dout, a.dim, sizeof(T), MOST);
  const int w = sb_vector_width(a.dtable, a.ld_dtable, a.dim, 4, v > 4 ? 4 : v);
  if (w < (v > 4 ? 4 : v)) v = w;
  if (v == 8) return launch_grad<T, MOST>(a, s);
  if (v == 4) return launch_grad<T, 4>(a, s);
  if (v == 2) return launch_grad<T, 2>(a, s);
  return launch_grad<T, 1>(a, s);
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
  *bytes = grad_plan(n, vocab, dim).bytes;
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
  const GradPlan p = grad_plan(n, vocab, dim);
  char* ws = (char*)workspace;
  SortArgs a;
  memset(&a, 0, sizeof(a));
  a.tokens = tokens; a.index64 = index_dtype == SB_I64;
  a.counts = (int*)(ws + p.counts); a.totals = (int*)(ws + p.totals);
  a.n = (int)n; a.vocab = vocab; a.bits = p.sort.bits; a.chunks = p.sort.chunks; a.chunk = p.sort.chunk;
  int* keys = (int*)(ws + p.keys);
  int* pos = (int*)(ws + p.pos);
  for (int pass = 0; pass < p.sort.passes; ++pass) {
    a.shift = pass * p.sort.bits;
    a.keys_in = keys + (pass & 1 ? 0 : n); a.pos_in = pos + (pass & 1 ? 0 : n);
    a.keys_out = keys + (pass & 1 ? n : 0); a.pos_out = pos + (pass & 1 ? n : 0);
    rc = pass == 0 ? launch_sort_pass<true>(a, p.sort, s) : launch_sort_pass<false>(a, p.sort, s);
    if (rc != SB_OK) return rc;
  }
  GradArgs g;
  memset(&g, 0, sizeof(g));
  g.keys = a.keys_out; g.pos = a.pos_out; g.dout = dout; g.dtable = dtable;
  g.carry = (float*)(ws + p.carry); g.run_key = (int*)(ws + p.run_key);
  g.ld_dout = ld_dout; g.ld_dtable = ld_dtable; g.n = (int)n; g.vocab = vocab; g.dim = dim;
  g.run_len = p.run_len; g.runs = p.runs; g.scale = scale; g.accumulate = accumulate;
  rc = dout_dtype == SB_F32 ? launch_grad_type<float>(g, s)
       : dout_dtype == SB_BF16 ? launch_grad_type<__nv_bfloat16>(g, s) : launch_grad_type<__half>(g, s);
  if (rc != SB_OK) return rc;
  if (p.runs > 1) {
    SB_CUDA(sb_launch(embedding_join_kernel, dim3(p.runs - 1), dim3(256), 0, s, 1, g));
    SB_COUNT_LAUNCH();
  }
  return SB_OK;
}

}  // extern "C"
