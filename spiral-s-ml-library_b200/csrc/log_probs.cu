// Log probabilities of given tokens under row distributions, their entropy and likeliest alternatives, and the gradient: what
// a policy gradient needs of a policy head, or a token loss of a large vocabulary.
//
// With s the scale (one over the temperature), x a row's legal logits, M their largest and S = sum exp(s (x_j - M)):
//   log p_j = s (x_j - M) - log S        H = log S - s sum exp(s (x_j - M)) (x_j - M) / S
//   d x_j = s (a ([j = t] - p_j) - h p_j (log p_j + H))      for the gradients a of log p_t and h of H.
#include "common.cuh"
#include "vector_io.cuh"

namespace {

constexpr int LP_MAX_TOP = 64;

struct LogProbArgs {
  const void* logits;
  long long ld, rows;
  int cols;                      // legal columns end here (the prefix), <= mask_cols
  int mask_cols;
  const uint8_t* mask;
  float scale;
  const void* tokens;
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

constexpr float LP_LOWEST = -3.402823466e38f;
// What a distance from the largest logit counts as at least where it is multiplied by its own probability: 0, not NaN, for -inf.
constexpr float LP_FAR = -1e30f;

template <typename T>
__device__ __forceinline__ float lp_logit(const LogProbArgs& g, long long row, int j) {
  const float x = sb_to_f32<T>(reinterpret_cast<const T*>(g.logits)[row * g.ld + j]);
  return g.mask && g.mask[row * g.mask_cols + j] == 0 ? -INFINITY : x;
}

template <typename I>
__device__ __forceinline__ long long lp_token(const void* tokens, long long row) { return (long long)reinterpret_cast<const I*>(tokens)[row]; }

// One block per row, the row read three times and once more per alternative.
template <typename T, typename I>
__global__ void __launch_bounds__(256) log_probs_kernel(LogProbArgs g) {
  __shared__ float part[8];
  __shared__ float part2[8];
  __shared__ int place[8];
  sb_grid_dependency_wait();
  sb_grid_dependents_launch();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (long long row = blockIdx.x; row < g.rows; row += gridDim.x) {
    float top = LP_LOWEST;
    for (int j = threadIdx.x; j < g.cols; j += 256) top = max_nan(top, lp_logit<T>(g, row, j));
    for (int o = 16; o; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
    __syncthreads();
    if (lane == 0) part[warp] = top;
    __syncthreads();
    for (int w = 0; w < 8; ++w) top = max_nan(top, part[w]);
    float sum = 0.f, dist = 0.f;
    for (int j = threadIdx.x; j < g.cols; j += 256) {
      const float d = max_nan(lp_logit<T>(g, row, j) - top, LP_FAR);
      const float e = __expf(d * g.scale);
      sum += e;
      dist += e * d;
    }
    for (int o = 16; o; o >>= 1) {
      sum += __shfl_xor_sync(0xffffffffu, sum, o);
      dist += __shfl_xor_sync(0xffffffffu, dist, o);
    }
    __syncthreads();
    if (lane == 0) { part[warp] = sum; part2[warp] = dist; }
    __syncthreads();
    sum = dist = 0.f;
    for (int w = 0; w < 8; ++w) { sum += part[w]; dist += part2[w]; }
    const bool empty = sum == 0.f;
    const float log_sum = empty ? INFINITY : logf(sum);
    if (threadIdx.x == 0) {
      if (g.out) {
        const long long t = lp_token<I>(g.tokens, row);
        g.out[row] = t < 0 || t >= g.mask_cols ? 0.f : t >= g.cols || empty ? -INFINITY : g.scale * (lp_logit<T>(g, row, (int)t) - top) - log_sum;
      }
      if (g.entropy) g.entropy[row] = empty ? 0.f : log_sum - g.scale * (dist / sum);
      if (g.stats) {
        g.stats[2 * row] = empty ? 0.f : top;
        g.stats[2 * row + 1] = log_sum;
      }
    }
    float last = INFINITY;
    int last_at = -1;
    for (int i = 0; i < g.top; ++i) {
      float best = -INFINITY;
      int at = 0x7fffffff;
      for (int j = threadIdx.x; j < g.cols; j += 256) {
        const float x = lp_logit<T>(g, row, j);
        if ((x < last || (x == last && j > last_at)) && x > best) { best = x; at = j; }
      }
      for (int o = 16; o; o >>= 1) {
        const float b = __shfl_xor_sync(0xffffffffu, best, o);
        const int a = __shfl_xor_sync(0xffffffffu, at, o);
        if (b > best || (b == best && a < at)) { best = b; at = a; }
      }
      __syncthreads();
      if (lane == 0) { part[warp] = best; place[warp] = at; }
      __syncthreads();
      for (int w = 0; w < 8; ++w)
        if (part[w] > best || (part[w] == best && place[w] < at)) { best = part[w]; at = place[w]; }
      const bool none = at == 0x7fffffff;
      if (threadIdx.x == 0) {
        if (g.top_values) g.top_values[row * g.top + i] = none ? -INFINITY : g.scale * (best - top) - log_sum;
        if (g.top_tokens) g.top_tokens[row * g.top + i] = none ? -1 : at;
      }
      last = best;
      last_at = at;
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
  const float* stats;
  const float* dout;
  const float* entropy;
  const float* dentropy;
};

template <typename T, typename I>
__global__ void __launch_bounds__(256) log_probs_grad_kernel(LogProbGradArgs g) {
  sb_grid_dependency_wait();
  sb_grid_dependents_launch();
  for (long long row = blockIdx.x; row < g.rows; row += gridDim.x) {
    const float top = g.stats[2 * row], log_sum = g.stats[2 * row + 1];
    long long t = g.dout ? lp_token<I>(g.tokens, row) : -1;
    const float a = t >= 0 && t < g.mask_cols ? g.dout[row] : 0.f;
    const float h = g.dentropy ? g.dentropy[row] : 0.f, entropy = g.dentropy ? g.entropy[row] : 0.f;
    if (log_sum == INFINITY) t = -1;
    for (int j = threadIdx.x; j < g.mask_cols; j += 256) {
      float d = 0.f;
      if (j < g.cols && !(g.mask && g.mask[row * g.mask_cols + j] == 0)) {
        const float x = sb_to_f32<T>(reinterpret_cast<const T*>(g.logits)[row * g.ld + j]);
        const float lp = max_nan(g.scale * (x - top) - log_sum, LP_FAR);
        const float p = __expf(lp);
        d = g.scale * ((j == t ? a : 0.f) - p * (a + h * (lp + entropy)));
      }
      reinterpret_cast<T*>(g.dlogits)[row * g.ldd + j] = sb_from_f32<T>(d);
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

template <typename T>
int launch_log_probs(const LogProbArgs& g, int index_dtype, cudaStream_t s) {
  const int grid = (int)(g.rows < 65536 ? g.rows : 65536);
  if (index_dtype == SB_I64) SB_CUDA(sb_launch(log_probs_kernel<T, long long>, dim3(grid), dim3(256), 0, s, 1, g));
  else SB_CUDA(sb_launch(log_probs_kernel<T, int>, dim3(grid), dim3(256), 0, s, 1, g));
  SB_COUNT_LAUNCH();
  return SB_OK;
}

template <typename T>
int launch_log_probs_grad(const LogProbGradArgs& g, int index_dtype, cudaStream_t s) {
  const int grid = (int)(g.rows < 65536 ? g.rows : 65536);
  if (index_dtype == SB_I64) SB_CUDA(sb_launch(log_probs_grad_kernel<T, long long>, dim3(grid), dim3(256), 0, s, 1, g));
  else SB_CUDA(sb_launch(log_probs_grad_kernel<T, int>, dim3(grid), dim3(256), 0, s, 1, g));
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
  g.mask = prefix >= 0 ? nullptr : mask; g.scale = scale; g.tokens = tokens; g.out = out; g.entropy = entropy; g.stats = stats;
  g.top = top; g.top_values = top_values; g.top_tokens = top_tokens;
  cudaStream_t s = (cudaStream_t)stream;
  return dtype == SB_F32 ? launch_log_probs<float>(g, index_dtype, s)
         : dtype == SB_BF16 ? launch_log_probs<__nv_bfloat16>(g, index_dtype, s) : launch_log_probs<__half>(g, index_dtype, s);
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
  g.mask = prefix >= 0 ? nullptr : mask; g.scale = scale; g.tokens = tokens; g.stats = stats; g.dout = dout; g.entropy = entropy;
  g.dentropy = dentropy; g.dlogits = dlogits; g.ldd = ldd;
  cudaStream_t s = (cudaStream_t)stream;
  return dtype == SB_F32 ? launch_log_probs_grad<float>(g, index_dtype, s)
         : dtype == SB_BF16 ? launch_log_probs_grad<__nv_bfloat16>(g, index_dtype, s) : launch_log_probs_grad<__half>(g, index_dtype, s);
}

}  // extern "C"
