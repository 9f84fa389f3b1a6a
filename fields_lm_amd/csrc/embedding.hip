// embedding.hip — rows of an embedding by token, scaled, and the gradient of its weight: with a scale s and the
// tokens k_n,
//   out[n] = s W[k_n],    dW[v] = s sum over n with k_n = v of g[n], in the order of n.
#include "fl_common.h"

namespace {

using namespace fl;

constexpr int64_t kMaxTokens = (int64_t)1 << 31, kMaxVocab = (int64_t)1 << 31, kMaxDim = (int64_t)1 << 24;

// 8 values at any element's address, `left` of them there
template <typename T>
__device__ __forceinline__ void load8(const T* p, int64_t left, float* v) {
  if (left >= 8) {
    if constexpr (sizeof(T) == 4) {
      const u32x4 a = *reinterpret_cast<const u32x4_any*>(p), b = *reinterpret_cast<const u32x4_any*>(p + 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[i] = __uint_as_float(a[i]);
        v[4 + i] = __uint_as_float(b[i]);
      }
    } else {
      const u32x4 a = *reinterpret_cast<const u32x4_any*>(p);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[2 * i] = bf16_lo(a[i]);
        v[2 * i + 1] = bf16_hi(a[i]);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < left ? load_as<T>(p + i) : 0.f;
  }
}

template <typename T>
__device__ __forceinline__ void store8(T* p, int64_t left, const float* v) {
  if (left >= 8) {
    if constexpr (sizeof(T) == 4) {
      u32x4 a, b;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        a[i] = __float_as_uint(v[i]);
        b[i] = __float_as_uint(v[4 + i]);
      }
      *reinterpret_cast<u32x4_any*>(p) = a;
      *reinterpret_cast<u32x4_any*>(p + 4) = b;
    } else {
      u32x4 a;
#pragma unroll
      for (int i = 0; i < 4; ++i) a[i] = bf16_pair(v[2 * i], v[2 * i + 1]);
      *reinterpret_cast<u32x4_any*>(p) = a;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) store_as(p + i, v[i]);
  }
}

// `lanes` lanes (a power of two) to a row, 8 values a lane and turn. MASKED: the transpose of the gradient, whose rows
// of `padding` and of tokens outside the vocabulary are zeros; else those of the latter are NaN.
template <typename WT, typename OT, bool MASKED>
__global__ __launch_bounds__(256) void fl_embedding_kernel(const int64_t* __restrict__ tokens, int64_t n,
                                                           const WT* __restrict__ weight, int64_t V, int64_t D,
                                                           int64_t stride, int lanes, int64_t padding, float scale,
                                                           OT* __restrict__ out) {
  const int64_t row = ((int64_t)blockIdx.x * 256 + threadIdx.x) / (unsigned)lanes;
  if (row >= n) return;
  const int64_t token = tokens[row];
  const bool inside = token >= 0 && token < V;
  const bool read = inside && !(MASKED && token == padding);
  const float other = MASKED ? 0.f : __uint_as_float(0x7fc00000u);
  const WT* w = weight + (read ? token : 0) * stride;
  for (int64_t c = (int64_t)(threadIdx.x & (lanes - 1)) * 8; c < D; c += (int64_t)lanes * 8) {
    float v[8];
    if (read) {
      load8(w + c, D - c, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] *= scale;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = other;
    }
    store8(out + row * D + c, D - c, v);
  }
}

// A wave to a row of the gradient and 512 columns: it looks through all tokens, 64 at a time, and adds the rows of
// those that are its own, in their order.
template <typename GT, typename WT>
__global__ __launch_bounds__(256) void fl_embedding_grad_kernel(const int64_t* __restrict__ tokens, int64_t n,
                                                                const GT* __restrict__ g, int64_t V, int64_t D,
                                                                int64_t padding, float scale, WT* __restrict__ out) {
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + uniform(threadIdx.x >> 6);
  if (row >= V) return;
  for (int64_t c = (int64_t)lane * 8; c - (int64_t)lane * 8 < D; c += 512) {
    float acc[8] = {};
    if (row != padding) {
      for (int64_t at = 0; at < n; at += 64) {
        uint64_t mine = __ballot(at + lane < n && tokens[at + lane < n ? at + lane : n - 1] == row);
        while (mine) {
          const int i = __ffsll((unsigned long long)mine) - 1;
          mine &= mine - 1;
          float v[8];
          if (c < D) {
            load8(g + (at + i) * D + c, D - c, v);
#pragma unroll
            for (int j = 0; j < 8; ++j) acc[j] += v[j];
          }
        }
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] *= scale;
    if (c < D) store8(out + row * D + c, D - c, acc);
  }
}

template <typename WT, typename OT>
int embedding(const int64_t* tokens, int64_t n, const void* weight, int64_t V, int64_t D, int64_t stride, int masked,
              int64_t padding, float scale, void* out, hipStream_t s) {
  int lanes = 1;
  while (lanes < 64 && lanes * 8 < D) lanes *= 2;
  const unsigned blocks = (unsigned)cdiv(n, 256 / lanes);
  if (masked)
    fl_embedding_kernel<WT, OT, true><<<blocks, 256, 0, s>>>(tokens, n, static_cast<const WT*>(weight), V, D, stride,
                                                              lanes, padding, scale, static_cast<OT*>(out));
  else
    fl_embedding_kernel<WT, OT, false><<<blocks, 256, 0, s>>>(tokens, n, static_cast<const WT*>(weight), V, D, stride,
                                                               lanes, padding, scale, static_cast<OT*>(out));
  return hip_status(hipGetLastError());
}

template <typename GT, typename WT>
int embedding_grad(const int64_t* tokens, int64_t n, const void* g, int64_t V, int64_t D, int64_t padding, float scale,
                   void* out, hipStream_t s) {
  fl_embedding_grad_kernel<GT, WT><<<(unsigned)cdiv(V, 4), 256, 0, s>>>(tokens, n, static_cast<const GT*>(g), V, D,
                                                                        padding, scale, static_cast<WT*>(out));
  return hip_status(hipGetLastError());
}

bool sizes_ok(int64_t n, int64_t V, int64_t D) {
  return n >= 0 && n <= kMaxTokens && V > 0 && V <= kMaxVocab && D > 0 && D <= kMaxDim;
}

}  // namespace

extern "C" {

int fl_embedding(const int64_t* tokens, int64_t n, const void* weight, int weight_dtype, int64_t V, int64_t D,
                 int64_t weight_stride, float scale, int masked, int64_t padding, void* out, int out_dtype,
                 void* stream) {
  if (!dtype_ok(weight_dtype) || !dtype_ok(out_dtype)) return FL_ERR_DTYPE;
  if (!sizes_ok(n, V, D) || weight_stride < 0) return FL_ERR_INVALID_ARGUMENT;
  if (n == 0) return FL_OK;
  if (!tokens || !weight || !out || !aligned(tokens, 8) || !aligned(weight, esize(weight_dtype)) ||
      !aligned(out, esize(out_dtype)))
    return FL_ERR_INVALID_ARGUMENT;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool w16 = weight_dtype == FL_DTYPE_BF16, o16 = out_dtype == FL_DTYPE_BF16;
  const auto call = w16 ? (o16 ? embedding<bf16_bits, bf16_bits> : embedding<bf16_bits, float>)
                        : (o16 ? embedding<float, bf16_bits> : embedding<float, float>);
  return call(tokens, n, weight, V, D, weight_stride, masked, padding, scale, out, s);
}

size_t fl_embedding_backward_workspace_bytes(int64_t n, int64_t V, int64_t D) {
  if (!sizes_ok(n, V, D)) return 0;
  return 16;
}

int fl_embedding_backward(const int64_t* tokens, int64_t n, const void* g, int g_dtype, int64_t V, int64_t D,
                          int64_t padding, float scale, void* g_weight, int weight_dtype, void* workspace,
                          size_t workspace_bytes, void* stream) {
  if (!dtype_ok(weight_dtype) || !dtype_ok(g_dtype)) return FL_ERR_DTYPE;
  if (!sizes_ok(n, V, D)) return FL_ERR_INVALID_ARGUMENT;
  if ((n && (!tokens || !g)) || !g_weight || !aligned(tokens, 8) || !aligned(g, esize(g_dtype)) ||
      !aligned(g_weight, esize(weight_dtype)))
    return FL_ERR_INVALID_ARGUMENT;
  if (!workspace || workspace_bytes < fl_embedding_backward_workspace_bytes(n, V, D)) return FL_ERR_WORKSPACE;
  if (!aligned(workspace, 16)) return FL_ERR_INVALID_ARGUMENT;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool w16 = weight_dtype == FL_DTYPE_BF16, g16 = g_dtype == FL_DTYPE_BF16;
  const auto call = g16 ? (w16 ? embedding_grad<bf16_bits, bf16_bits> : embedding_grad<bf16_bits, float>)
                        : (w16 ? embedding_grad<float, bf16_bits> : embedding_grad<float, float>);
  return call(tokens, n, g, V, D, padding, scale, g_weight, s);
}

}  // extern "C"
