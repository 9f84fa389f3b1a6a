// logprobs.hip — log probabilities of given tokens with entropy and top alternatives, and their gradient.
//
// For a row x of V logits, temperature T and token t: with m = max x and d_v = (x_v - m) / T,
//   lp = d_t - ln s,  s = sum e^{d_v};   H = ln s - (sum e^{d_v} d_v) / s;   the K largest x and their lp.
// Gradient, from g of lp, h of H and g_k of the alternatives i_k, p_v = e^{d_v - ln s}:
//   dx_v = ([v = t] g + sum_k [v = i_k] g_k - p_v (g + sum_k g_k) - h p_v (ln p_v + H)) / T.
// d and ln s are kept apart, so that large logits lose nothing, and nothing is divided before the maximum is
// subtracted, so that masks of the type's lowest value stay finite.
#include "fl_common.h"

namespace {

using namespace fl;

constexpr int kMaxTop = 64;
constexpr float kLn2 = 0.6931471805599453f;

struct Rows {
  int64_t inner;                      // row r is (r / inner, r % inner)
  int64_t stride_outer, stride_inner; // of the logits, in elements
  int64_t token_outer, token_inner;   // of the tokens
  __device__ __forceinline__ int64_t logits(int64_t r) const { return r / inner * stride_outer + r % inner * stride_inner; }
  __device__ __forceinline__ int64_t token(int64_t r) const { return r / inner * token_outer + r % inner * token_inner; }
};

// Order of the alternatives as an integer: larger values first, -0 as 0, NaN above all, then the lower index.
// Every key lies strictly between 0 and ~0, which stand for none and for no limit.
__device__ __forceinline__ uint64_t rank_key(float x, uint32_t index) {
  uint32_t b = __float_as_uint(x + 0.0f);
  b = b & 0x80000000u ? ~b : b | 0x80000000u;
  if (x != x) b = 0xfffffffeu;
  return (uint64_t)b << 32 | (0xffffffffu - index);
}

template <typename V, typename Op>
__device__ __forceinline__ V block_reduce(V v, V* s, Op op) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) v = op(v, __shfl_xor(v, d));
  __syncthreads();  // s may still be read from the last reduction
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
  __syncthreads();
  v = s[0];
  for (int i = 1; i < (int)(blockDim.x >> 6); ++i) v = op(v, s[i]);
  return v;
}

__device__ __forceinline__ float quiet_nan() { return __uint_as_float(0x7fc00000u); }

// One block to a row.
template <typename T>
__global__ __launch_bounds__(256) void fl_token_logprobs_kernel(
    const T* __restrict__ logits, Rows rows, int64_t n_rows, int V, const int64_t* __restrict__ tokens,
    int64_t ignore, float inv_t, int K, float* __restrict__ logprobs, float* __restrict__ entropy,
    float* __restrict__ top_lp, int64_t* __restrict__ top_tok, float* __restrict__ stats) {
  __shared__ float s_f[4];
  __shared__ unsigned long long s_k[4];
  for (int64_t row = blockIdx.x; row < n_rows; row += gridDim.x) {
    const T* x = logits + rows.logits(row);
    float top = -INFINITY, sum = 0.f, ent = 0.f;
    bool nan = false;
    for (int i = threadIdx.x; i < V; i += 256) {
      const float v = load_as<T>(x + i);
      nan |= v != v;
      top = fmaxf(top, v);
    }
    top = block_reduce(nan ? INFINITY : top, s_f, [](float a, float b) { return fmaxf(a, b); });
    const bool empty = top == -INFINITY;
    const float base = empty ? 0.f : top;
    for (int i = threadIdx.x; i < V; i += 256) {
      const float d = (load_as<T>(x + i) - base) * inv_t, e = __builtin_amdgcn_exp2f(d * kLog2e);
      sum += e;
      if (e > 0.f) ent = fmaf(e, d, ent);
    }
    const auto add = [](float a, float b) { return a + b; };
    sum = block_reduce(sum, s_f, add);
    ent = block_reduce(ent, s_f, add);
    const float log_sum = __builtin_amdgcn_logf(sum) * kLn2;
    const auto lp_of = [&](float v) { return empty ? -INFINITY : (v - base) * inv_t - log_sum; };
    if (threadIdx.x == 0) {
      const int64_t t = tokens[rows.token(row)];
      logprobs[row] = t == ignore ? 0.f : t >= 0 && t < V ? lp_of(load_as<T>(x + t)) : quiet_nan();
      if (entropy) entropy[row] = empty ? 0.f : log_sum - ent / sum;
      if (stats) {
        stats[2 * row] = top;
        stats[2 * row + 1] = log_sum;
      }
    }
    unsigned long long last = ~0ull;
    for (int k = 0; k < K; ++k) {
      unsigned long long best = 0;
      for (int i = threadIdx.x; i < V; i += 256) {
        const unsigned long long key = rank_key(load_as<T>(x + i), (uint32_t)i);
        if (key < last && key > best) best = key;
      }
      last = block_reduce(best, s_k, [](unsigned long long a, unsigned long long b) { return a > b ? a : b; });
      if (threadIdx.x == 0) {
        const uint32_t at = 0xffffffffu - (uint32_t)last;
        top_tok[row * K + k] = at;
        top_lp[row * K + k] = lp_of(load_as<T>(x + at));
      }
    }
  }
}

// Gradient of one row by one block. A row whose gradients are all 0 gets zeros whatever its logits hold.
template <typename T>
__global__ __launch_bounds__(256) void fl_token_logprobs_backward_kernel(
    const T* __restrict__ logits, Rows rows, int64_t n_rows, int V, const int64_t* __restrict__ tokens,
    int64_t ignore, float inv_t, int K, const float* __restrict__ stats, const float* __restrict__ entropy,
    const int64_t* __restrict__ top_tok, const float* __restrict__ g_lp, const float* __restrict__ g_ent,
    const float* __restrict__ g_top, T* __restrict__ grad) {
  for (int64_t row = blockIdx.x; row < n_rows; row += gridDim.x) {
    const T* x = logits + rows.logits(row);
    T* out = grad + row * V;
    const int64_t t = tokens[rows.token(row)];
    float g = g_lp && t != ignore ? g_lp[row] : 0.f;
    const float h = g_ent ? g_ent[row] : 0.f;
    float a = g;
    bool any = g != 0.f || h != 0.f;
    for (int k = 0; k < (g_top ? K : 0); ++k) {
      const float gk = g_top[row * K + k];
      a += gk;
      any |= gk != 0.f;
    }
    const float top = stats[2 * row], log_sum = stats[2 * row + 1];
    if (!any || top == -INFINITY) {
      for (int i = threadIdx.x; i < V; i += 256) store_as(out + i, 0.f);
      continue;
    }
    if (g != 0.f && (t < 0 || t >= V)) a = quiet_nan();
    const float ent = h != 0.f ? entropy[row] : 0.f;
    const auto part = [&](float v) {  // -p (a + h (ln p + H))
      const float lp = (v - top) * inv_t - log_sum, p = __builtin_amdgcn_exp2f(lp * kLog2e);
      const float w = h != 0.f && p > 0.f ? fmaf(h, lp + ent, a) : a;
      return -p * w;
    };
    for (int i = threadIdx.x; i < V; i += 256) {
      float v = part(load_as<T>(x + i));
      if (i == t) v += g;
      for (int k = 0; k < (g_top ? K : 0); ++k)
        if (i == top_tok[row * K + k]) v += g_top[row * K + k];
      store_as(out + i, v * inv_t);
    }
  }
}

constexpr int64_t kMaxBlocks = 1 << 20;

bool shape_ok(int64_t outer, int64_t inner, int64_t V, int64_t so, int64_t si) {
  return outer > 0 && inner > 0 && outer <= ((int64_t)1 << 40) / inner && V > 0 && V < ((int64_t)1 << 31) && so >= 0 && si >= 0;
}

}  // namespace

extern "C" {

size_t fl_token_logprobs_workspace_bytes(int64_t rows, int64_t V, int64_t top_k) {
  (void)rows;
  (void)V;
  (void)top_k;
  return 0;
}

int fl_token_logprobs(const void* logits, int dtype, int64_t outer, int64_t inner, int64_t V, int64_t stride_outer,
                      int64_t stride_inner, const int64_t* tokens, int64_t token_outer, int64_t token_inner,
                      int64_t ignore_index, float temperature, int64_t top_k, float* logprobs, float* entropy,
                      float* top_logprobs, int64_t* top_tokens, float* stats, void* workspace, size_t workspace_bytes,
                      void* stream) {
  if (!dtype_ok(dtype)) return FL_ERR_DTYPE;
  if (!shape_ok(outer, inner, V, stride_outer, stride_inner) || !(temperature > 0.f) || !(1.0f / temperature > 0.f) ||
      top_k < 0 || top_k > kMaxTop || top_k > V)
    return FL_ERR_INVALID_ARGUMENT;
  if (!logits || !aligned(logits, esize(dtype)) || !tokens || !aligned(tokens, 8) || !logprobs || !aligned(logprobs, 4) ||
      !aligned(entropy, 4) || !aligned(stats, 4) ||
      (top_k && (!top_logprobs || !top_tokens || !aligned(top_logprobs, 4) || !aligned(top_tokens, 8))))
    return FL_ERR_INVALID_ARGUMENT;
  (void)workspace;
  (void)workspace_bytes;
  const int64_t rows = outer * inner;
  const Rows r = {inner, stride_outer, stride_inner, token_outer, token_inner};
  const unsigned blocks = (unsigned)(rows < kMaxBlocks ? rows : kMaxBlocks);
  hipStream_t s = static_cast<hipStream_t>(stream);
#define FL_LP(T)                                                                                                  \
  fl_token_logprobs_kernel<T><<<blocks, 256, 0, s>>>(static_cast<const T*>(logits), r, rows, (int)V, tokens,      \
                                                     ignore_index, 1.0f / temperature, (int)top_k, logprobs,      \
                                                     entropy, top_logprobs, top_tokens, stats)
  if (dtype == FL_DTYPE_BF16) FL_LP(bf16_bits);
  else FL_LP(float);
#undef FL_LP
  return hip_status(hipGetLastError());
}

int fl_token_logprobs_backward(const void* logits, int dtype, int64_t outer, int64_t inner, int64_t V,
                               int64_t stride_outer, int64_t stride_inner, const int64_t* tokens, int64_t token_outer,
                               int64_t token_inner, int64_t ignore_index, float temperature, int64_t top_k,
                               const float* stats, const float* entropy, const int64_t* top_tokens,
                               const float* g_logprobs, const float* g_entropy, const float* g_top, void* g_logits,
                               void* stream) {
  if (!dtype_ok(dtype)) return FL_ERR_DTYPE;
  if (!shape_ok(outer, inner, V, stride_outer, stride_inner) || !(temperature > 0.f) || !(1.0f / temperature > 0.f) ||
      top_k < 0 || top_k > kMaxTop || top_k > V)
    return FL_ERR_INVALID_ARGUMENT;
  if (!logits || !aligned(logits, esize(dtype)) || !tokens || !aligned(tokens, 8) || !stats || !aligned(stats, 4) ||
      !g_logits || !aligned(g_logits, esize(dtype)) || !aligned(g_logprobs, 4) || !aligned(g_entropy, 4) ||
      !aligned(g_top, 4) || (g_entropy && (!entropy || !aligned(entropy, 4))) ||
      (g_top && (top_k == 0 || !top_tokens || !aligned(top_tokens, 8))))
    return FL_ERR_INVALID_ARGUMENT;
  const int64_t rows = outer * inner;
  const Rows r = {inner, stride_outer, stride_inner, token_outer, token_inner};
  const unsigned blocks = (unsigned)(rows < kMaxBlocks ? rows : kMaxBlocks);
  hipStream_t s = static_cast<hipStream_t>(stream);
#define FL_LB(T)                                                                                                    \
  fl_token_logprobs_backward_kernel<T><<<blocks, 256, 0, s>>>(                                                      \
      static_cast<const T*>(logits), r, rows, (int)V, tokens, ignore_index, 1.0f / temperature, (int)top_k, stats,  \
      entropy, top_tokens, g_logprobs, g_entropy, g_top, static_cast<T*>(g_logits))
  if (dtype == FL_DTYPE_BF16) FL_LB(bf16_bits);
  else FL_LB(float);
#undef FL_LB
  return hip_status(hipGetLastError());
}

}  // extern "C"
