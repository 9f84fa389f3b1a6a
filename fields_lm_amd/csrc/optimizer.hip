// optimizer.hip — what follows a training step's backward, over many tensors at once: the 2-norm of all
// gradients with the scale that clips it, and the AdamW step, its moments in fp32 or in 8 bits.
//
// The tensors' addresses travel in the kernel arguments (kTensors to a launch), so that a call copies nothing
// to the device and can be captured; blocks find their tensor by the running count of blocks. Sums are taken
// in a fixed order.
//
// Compiled without contraction: the 8-bit codes next to a border between two go by the bits of the moments,
// which are those of separate products and sums.
#include "fl_common.h"

namespace {

using namespace fl;

constexpr int kTensors = 64;      // tensors of a launch (an 8-bit table of 64 is 3.6 KiB of arguments)
constexpr int kStepTensors = 256; // step counters of a launch
constexpr int kChunk = 4096;      // values of a block
constexpr int kBlock = 256;       // values that share a scale in the 8-bit states
constexpr int kMaxBlocks = 1 << 23;  // blocks of a launch

// 8-bit states: a block's largest magnitude takes e4m3's largest code; a block below kTiny is held as zeros
constexpr float kTopCode = 448.0f, kSmallest = 0.001953125f, kTiny = 1e-30f;

struct NormTable {
  const void* x[kTensors];
  int64_t numel[kTensors];
  int first[kTensors + 1];  // running count of blocks
  int is_bf16[kTensors];
  int n;
};

template <bool EIGHT>
struct AdamTable {
  void* p[kTensors];
  const void* g[kTensors];
  void* m[kTensors];
  void* v[kTensors];
  float* ms[EIGHT ? kTensors : 1];
  float* vs[EIGHT ? kTensors : 1];
  int64_t numel[kTensors];
  int first[kTensors + 1];
  int n;
};

struct StepTable {
  int64_t* step[kStepTensors];
  int n;
};

template <typename Table>
__device__ __forceinline__ int tensor_of(const Table& t, int block) {
  int i = 0;
  while (i + 1 < t.n && t.first[i + 1] <= block) ++i;
  return i;
}

template <typename T>
__device__ double square_sum(const T* x, int64_t lo, int64_t hi) {
  double acc = 0.0;
  for (int64_t i = lo + threadIdx.x; i < hi; i += 256) {
    const double v = load_as<T>(x + i);
    acc = fma(v, v, acc);
  }
  return acc;
}

// sum over a block's threads, in thread 0
__device__ double block_sum(double v, double* s_sum) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
  if ((threadIdx.x & 63) == 0) s_sum[threadIdx.x >> 6] = v;
  __syncthreads();
  double t = 0.0;
  for (int i = 0; i < (int)blockDim.x / 64; ++i) t += s_sum[i];
  return t;
}

__global__ __launch_bounds__(256) void fl_square_sum_kernel(const NormTable t, double* __restrict__ part) {
  __shared__ double s_sum[4];
  const int i = tensor_of(t, (int)blockIdx.x);
  const int64_t lo = (int64_t)((int)blockIdx.x - t.first[i]) * kChunk, n = t.numel[i], hi = lo + kChunk < n ? lo + kChunk : n;
  const double v = t.is_bf16[i] ? square_sum(static_cast<const bf16_bits*>(t.x[i]), lo, hi)
                                : square_sum(static_cast<const float*>(t.x[i]), lo, hi);
  const double sum = block_sum(v, s_sum);
  if (threadIdx.x == 0) part[blockIdx.x] = sum;
}

// out[0] = the norm; out[1] = min(1, max_norm / (norm + 1e-6)), NaN for a norm that is not finite
__global__ __launch_bounds__(1024) void fl_norm_finish_kernel(const double* __restrict__ part, int64_t n, float max_norm,
                                                              float* __restrict__ out, int scaled) {
  __shared__ double s_sum[16];
  double acc = 0.0;
  for (int64_t i = threadIdx.x; i < n; i += 1024) acc += part[i];
  const double sum = block_sum(acc, s_sum);
  if (threadIdx.x == 0) {
    const float norm = (float)sqrt(sum);
    out[0] = norm;
    if (scaled) {
      const float s = max_norm / (norm + 1e-6f);
      out[1] = norm - norm == 0.0f ? (s < 1.0f ? s : 1.0f) : __uint_as_float(0x7fc00000u);
    }
  }
}

// A tensor's factors of this step: hyper = {lr / (1 - b1^t), (1 - b2^t)^-1/2, 1 - lr decay, gradient scale},
// and the step counted, or where the scale is not finite a scale of NaN and nothing counted.
__global__ __launch_bounds__(256) void fl_adamw_factors_kernel(const StepTable t, double lr, const float* lr_ptr,
                                                               double b1, double b2, double decay,
                                                               const float* __restrict__ grad_scale,
                                                               f32x4* __restrict__ hyper) {
  const int i = threadIdx.x;
  if (i >= t.n) return;
  const float gs = grad_scale ? *grad_scale : 1.0f;
  f32x4 h = {0.f, 0.f, 0.f, __uint_as_float(0x7fc00000u)};
  if (gs - gs == 0.0f) {
    const int64_t step = *t.step[i] + 1;
    *t.step[i] = step;
    const double rate = lr_ptr ? (double)*lr_ptr : lr;
    h[0] = (float)(rate / (1.0 - pow(b1, (double)step)));
    h[1] = (float)(1.0 / sqrt(1.0 - pow(b2, (double)step)));
    h[2] = (float)(1.0 - rate * decay);
    h[3] = gs;
  }
  hyper[i] = h;
}

struct Factors {
  float step, root_scale, decay, gs, b1, b1c, b2, b2c, eps;
};

// one value: m and v in, m, v and its root out; the new parameter
__device__ __forceinline__ float adamw_value(float p, float g, float& m, float& v, float& root, const Factors& f) {
  g = g * f.gs;
  m = m * f.b1 + g * f.b1c;
  v = v * f.b2 + (g * f.b2c) * g;
  root = sqrtf(v);
  return p * f.decay - f.step * (m / (root * f.root_scale + f.eps));
}

template <typename T>
__global__ __launch_bounds__(256) void fl_adamw_kernel(const AdamTable<false> t, const f32x4* __restrict__ hyper,
                                                       float b1, float b1c, float b2, float b2c, float eps) {
  const int i = tensor_of(t, (int)blockIdx.x);
  const f32x4 h = hyper[i];
  if (h[3] != h[3]) return;
  const Factors f = {h[0], h[1], h[2], h[3], b1, b1c, b2, b2c, eps};
  const int64_t lo = (int64_t)((int)blockIdx.x - t.first[i]) * kChunk, n = t.numel[i], hi = lo + kChunk < n ? lo + kChunk : n;
  T* p = static_cast<T*>(t.p[i]);
  const T* g = static_cast<const T*>(t.g[i]);
  float *ms = static_cast<float*>(t.m[i]), *vs = static_cast<float*>(t.v[i]);
  for (int64_t k = lo + threadIdx.x; k < hi; k += 256) {
    float m = ms[k], v = vs[k], root;
    store_as(p + k, adamw_value(load_as<T>(p + k), load_as<T>(g + k), m, v, root, f));
    ms[k] = m;
    vs[k] = v;
  }
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) v = fmaxf(v, __shfl_xor(v, d));
  return v;
}

// One wave to a block of 256 values. m is held as the e4m3 code of m (448 / max|m|), v as that of its root
// r (448 / max r), with max / 448 beside: a root keeps v's range in half the octaves, and one that is not 0
// keeps at least the smallest code, since a v that rounds to 0 under an m that does not would let the next
// step with a small gradient run away.
template <typename T>
__global__ __launch_bounds__(256) void fl_adamw8_kernel(const AdamTable<true> t, const f32x4* __restrict__ hyper,
                                                        float b1, float b1c, float b2, float b2c, float eps) {
  const int i = tensor_of(t, (int)blockIdx.x);
  const f32x4 h = hyper[i];
  if (h[3] != h[3]) return;
  const Factors f = {h[0], h[1], h[2], h[3], b1, b1c, b2, b2c, eps};
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t n = t.numel[i], lo = (int64_t)((int)blockIdx.x - t.first[i]) * kChunk;
  T* p = static_cast<T*>(t.p[i]);
  const T* g = static_cast<const T*>(t.g[i]);
  uint8_t *mc = static_cast<uint8_t*>(t.m[i]), *vc = static_cast<uint8_t*>(t.v[i]);
  for (int64_t at = lo + wave * kBlock; at < lo + kChunk && at < n; at += 4 * kBlock) {
    const int64_t b = at / kBlock;
    const float s_m = t.ms[i][b], s_v = t.vs[i][b];
    float m[4], r[4], top_m = 0.f, top_r = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t k = at + 4 * lane + j;
      m[j] = r[j] = 0.f;
      if (k < n) {
        m[j] = __builtin_amdgcn_cvt_f32_fp8((int)mc[k], 0) * s_m;
        const float root = __builtin_amdgcn_cvt_f32_fp8((int)vc[k], 0) * s_v;
        float v = root * root;
        store_as(p + k, adamw_value(load_as<T>(p + k), load_as<T>(g + k), m[j], v, r[j], f));
      }
      top_m = fmaxf(top_m, fabsf(m[j]));
      top_r = fmaxf(top_r, r[j]);
    }
    top_m = wave_max(top_m);
    top_r = wave_max(top_r);
    const float inv_m = top_m >= kTiny ? 1.0f / top_m * kTopCode : 0.f, inv_r = top_r >= kTiny ? 1.0f / top_r * kTopCode : 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t k = at + 4 * lane + j;
      float y = r[j] * inv_r;
      y = y > 0.f && y < kSmallest ? kSmallest : y;
      const int codes = __builtin_amdgcn_cvt_pk_fp8_f32(m[j] * inv_m, y, 0, false);
      if (k < n) {
        mc[k] = (uint8_t)codes;
        vc[k] = (uint8_t)(codes >> 8);
      }
    }
    if (lane == 0) {
      t.ms[i][b] = top_m >= kTiny ? top_m * (1.0f / kTopCode) : 0.f;
      t.vs[i][b] = top_r >= kTiny ? top_r * (1.0f / kTopCode) : 0.f;
    }
  }
}

constexpr int64_t kMaxNumel = (int64_t)1 << 34;  // 2^22 blocks: a tensor always fits a launch of 2^23
constexpr int64_t kMaxTensors = 1 << 20;

// Fills `table` with tensors from `i` on, empty ones too; returns the index after the last one taken.
template <typename Table, typename Put>
int64_t fill_table(Table& table, int64_t n, const int64_t* numel, int64_t i, Put put) {
  table.n = 0;
  table.first[0] = 0;
  for (; i < n && table.n < kTensors; ++i) {
    const int64_t blocks = cdiv(numel[i], kChunk);
    if (table.first[table.n] + blocks > kMaxBlocks) break;
    put(table.n, i);
    table.numel[table.n] = numel[i];
    table.first[table.n + 1] = table.first[table.n] + (int)blocks;
    ++table.n;
  }
  return i;
}

template <bool EIGHT, typename T>
int adamw_launch(int64_t n, void* const* params, const void* const* grads, void* const* m, void* const* v,
                 float* const* ms, float* const* vs, const int64_t* numel, const f32x4* hyper, double b1, double b2,
                 double eps, hipStream_t s) {
  const float c[5] = {(float)b1, (float)(1.0 - b1), (float)b2, (float)(1.0 - b2), (float)eps};
  for (int64_t i = 0; i < n;) {
    AdamTable<EIGHT> t = {};
    const f32x4* factors = hyper + i;
    i = fill_table(t, n, numel, i, [&](int k, int64_t j) {
      t.p[k] = params[j];
      t.g[k] = grads[j];
      t.m[k] = m[j];
      t.v[k] = v[j];
      if constexpr (EIGHT) {
        t.ms[k] = ms[j];
        t.vs[k] = vs[j];
      }
    });
    const unsigned blocks = (unsigned)t.first[t.n];
    if (blocks == 0) continue;
    if constexpr (EIGHT)
      fl_adamw8_kernel<T><<<blocks, 256, 0, s>>>(t, factors, c[0], c[1], c[2], c[3], c[4]);
    else
      fl_adamw_kernel<T><<<blocks, 256, 0, s>>>(t, factors, c[0], c[1], c[2], c[3], c[4]);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return hip_status(e);
  }
  return FL_OK;
}

bool list_ok(int64_t n, const int64_t* numel) {
  if (n <= 0 || n > kMaxTensors || !numel) return false;
  for (int64_t i = 0; i < n; ++i)
    if (numel[i] < 0 || numel[i] > kMaxNumel) return false;
  return true;
}

// every non-empty tensor has an address, a multiple of its elements' size
bool addresses_ok(int64_t n, const void* const* p, const int64_t* numel, size_t size) {
  if (!p) return false;
  for (int64_t i = 0; i < n; ++i)
    if (numel[i] > 0 && (!p[i] || !aligned(p[i], size))) return false;
  return true;
}

}  // namespace

extern "C" {

size_t fl_grad_norm_workspace_bytes(int64_t n, const int64_t* numel) {
  if (!list_ok(n, numel)) return 0;
  int64_t blocks = 0;
  for (int64_t i = 0; i < n; ++i) blocks += cdiv(numel[i], kChunk);
  return (size_t)(blocks > 0 ? blocks : 1) * sizeof(double);
}

int fl_grad_norm(int64_t n, const void* const* grads, const int* dtypes, const int64_t* numel, float max_norm, int scaled,
                 float* out, void* workspace, size_t workspace_bytes, void* stream) {
  if (!list_ok(n, numel) || !grads || !dtypes) return FL_ERR_INVALID_ARGUMENT;
  for (int64_t i = 0; i < n; ++i) {
    if (!dtype_ok(dtypes[i])) return FL_ERR_DTYPE;
    if (!addresses_ok(1, grads + i, numel + i, esize(dtypes[i]))) return FL_ERR_INVALID_ARGUMENT;
  }
  if (!out || !aligned(out, 4) || (scaled && !(max_norm >= 0.f))) return FL_ERR_INVALID_ARGUMENT;
  if (!workspace || workspace_bytes < fl_grad_norm_workspace_bytes(n, numel)) return FL_ERR_WORKSPACE;
  if (!aligned(workspace, 8)) return FL_ERR_INVALID_ARGUMENT;
  hipStream_t s = static_cast<hipStream_t>(stream);
  double* part = static_cast<double*>(workspace);
  int64_t done = 0;
  for (int64_t i = 0; i < n;) {
    NormTable t = {};
    i = fill_table(t, n, numel, i, [&](int k, int64_t j) {
      t.x[k] = grads[j];
      t.is_bf16[k] = dtypes[j] == FL_DTYPE_BF16;
    });
    const int blocks = t.first[t.n];
    if (blocks == 0) continue;
    fl_square_sum_kernel<<<(unsigned)blocks, 256, 0, s>>>(t, part + done);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return hip_status(e);
    done += blocks;
  }
  fl_norm_finish_kernel<<<1, 1024, 0, s>>>(part, done, max_norm, out, scaled);
  return hip_status(hipGetLastError());
}

size_t fl_adamw_workspace_bytes(int64_t n) { return n > 0 && n <= kMaxTensors ? (size_t)n * 16 : 0; }

int fl_adamw_step(int64_t n, void* const* params, const void* const* grads, int dtype, void* const* exp_avgs,
                  void* const* exp_avg_sqs, float* const* exp_avg_scales, float* const* exp_avg_sq_scales,
                  const int64_t* numel, int64_t* const* steps, double lr, const float* lr_ptr, double beta1, double beta2,
                  double eps, double weight_decay, const float* grad_scale, void* workspace, size_t workspace_bytes,
                  void* stream) {
  if (!dtype_ok(dtype)) return FL_ERR_DTYPE;
  const bool eight = exp_avg_scales != nullptr;
  if (!list_ok(n, numel) || eight != (exp_avg_sq_scales != nullptr)) return FL_ERR_INVALID_ARGUMENT;
  const size_t state = eight ? 1 : 4;
  if (!addresses_ok(n, (const void* const*)params, numel, esize(dtype)) ||
      !addresses_ok(n, grads, numel, esize(dtype)) ||
      !addresses_ok(n, (const void* const*)exp_avgs, numel, state) ||
      !addresses_ok(n, (const void* const*)exp_avg_sqs, numel, state) ||
      (eight && (!addresses_ok(n, (const void* const*)exp_avg_scales, numel, 4) ||
                 !addresses_ok(n, (const void* const*)exp_avg_sq_scales, numel, 4))))
    return FL_ERR_INVALID_ARGUMENT;
  if (!steps) return FL_ERR_INVALID_ARGUMENT;
  for (int64_t i = 0; i < n; ++i)
    if (!steps[i] || !aligned(steps[i], 8)) return FL_ERR_INVALID_ARGUMENT;
  if (!(beta1 >= 0.0 && beta1 < 1.0) || !(beta2 >= 0.0 && beta2 < 1.0) || !(eps >= 0.0) || !aligned(lr_ptr, 4) ||
      !aligned(grad_scale, 4))
    return FL_ERR_INVALID_ARGUMENT;
  if (!workspace || workspace_bytes < fl_adamw_workspace_bytes(n)) return FL_ERR_WORKSPACE;
  if (!aligned(workspace, 16)) return FL_ERR_INVALID_ARGUMENT;
  hipStream_t s = static_cast<hipStream_t>(stream);
  f32x4* hyper = static_cast<f32x4*>(workspace);
  for (int64_t i = 0; i < n; i += kStepTensors) {
    StepTable t = {};
    t.n = (int)(n - i < kStepTensors ? n - i : kStepTensors);
    for (int k = 0; k < t.n; ++k) t.step[k] = steps[i + k];
    fl_adamw_factors_kernel<<<1, 256, 0, s>>>(t, lr, lr_ptr, beta1, beta2, weight_decay, grad_scale, hyper + i);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return hip_status(e);
  }
#define FL_AW(E, T)                                                                                              \
  return adamw_launch<E, T>(n, params, grads, exp_avgs, exp_avg_sqs, exp_avg_scales, exp_avg_sq_scales, numel,   \
                            hyper, beta1, beta2, eps, s);
  const bool b16 = dtype == FL_DTYPE_BF16;
  if (eight && b16) FL_AW(true, bf16_bits)
  if (eight) FL_AW(true, float)
  if (b16) FL_AW(false, bf16_bits)
  FL_AW(false, float)
#undef FL_AW
}

}  // extern "C"
