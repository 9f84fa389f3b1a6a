// optimizer.hip — what follows a training step's backward, over many tensors at once: the 2-norm of all
// gradients with the scale that clips it, and the AdamW step, its moments in fp32 or in 8 bits.
//
// The tensors' addresses travel in the kernel arguments (kTensors, kNormTensors to a launch), so that a call copies
// nothing to the device and can be captured; blocks find their tensor by the running count of blocks. Sums are
// taken in a fixed order.
//
// Compiled without contraction: the 8-bit codes next to a border between two go by the bits of the moments,
// which are those of separate products and sums.
#include "fl_common.h"

namespace {

using namespace fl;

constexpr int kTensors = 64;      // tensors of a step's launch (an 8-bit table of 64 is 3.6 KiB of arguments)
constexpr int kNormTensors = 192;  // tensors of the norm's (3.8 KiB)
constexpr int kStepTensors = 480; // step counters of a launch, one to a thread
constexpr int kChunk = 2048;      // values of a step's block (the 8-bit step of 0.29 G bf16 values: 505 us; with 4,096
                                  // 522, with 1,024 544; the 32-bit step of as many fp32 1,415, 1,480 and 1,413)
constexpr int kBlock = 256;       // values that share a scale in the 8-bit states
constexpr int kMaxBlocks = 1 << 23;  // blocks of a launch

// 8-bit states: a block's largest magnitude takes e4m3's largest code; a block below kTiny is held as zeros
constexpr float kTopCode = 448.0f, kSmallest = 0.001953125f, kTiny = 1e-30f;

struct NormTable {
  static constexpr int kSize = kNormTensors;
  const void* x[kSize];
  int64_t numel[kSize];
  int first[kSize + 1];  // running count of blocks
  uint32_t is_bf16[kSize / 32];  // a bit to a tensor
  int n;
};

template <bool EIGHT>
struct AdamTable {
  static constexpr int kSize = kTensors;
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

// the tensor that `block` belongs to: as many end at or before it
template <typename Table>
__device__ __forceinline__ int tensor_of(const Table& t, int block) {
  const int lane = threadIdx.x & 63;
  int ended = 0;
#pragma unroll
  for (int i = 0; i < Table::kSize; i += 64)
    ended += __popcll(__ballot(i + lane < t.n && t.first[i + lane + 1] <= block));
  return ended;
}

// What a step touches once it touches past the caches' keeping (0.29 G values: the norm 204 us plain and 179
// streaming, the 32-bit step behind it 1,776 and 1,581 us in all, the 8-bit step 887 and 777; bf16 weights with 32-bit
// states alone lose, 1,166 and 1,207).
__device__ __forceinline__ u32x4 load_once(const u32x4_any* p) { return __builtin_nontemporal_load(p); }
__device__ __forceinline__ u32x2 load_once(const u32x2_any* p) { return __builtin_nontemporal_load(p); }
__device__ __forceinline__ uint32_t load_once(const u32_any* p) { return __builtin_nontemporal_load(p); }
__device__ __forceinline__ void store_once(u32x4_any* p, u32x4 v) { __builtin_nontemporal_store(v, p); }
__device__ __forceinline__ void store_once(u32x2_any* p, u32x2 v) { __builtin_nontemporal_store(v, p); }
__device__ __forceinline__ void store_once(u32_any* p, uint32_t v) { __builtin_nontemporal_store(v, p); }

// N consecutive values of an accessed 16 bytes, at any element's address
template <typename T>
struct Values;
template <>
struct Values<float> {
  static constexpr int N = 4;
  __device__ __forceinline__ static float get(const u32x4& r, int q) { return __uint_as_float(r[q]); }
};
template <>
struct Values<bf16_bits> {
  static constexpr int N = 8;
  __device__ __forceinline__ static float get(const u32x4& r, int q) {
    return q & 1 ? bf16_hi(r[q >> 1]) : bf16_lo(r[q >> 1]);
  }
};

// Four packs of 16 bytes a turn to a thread, each into a sum of its own.
template <typename T>
__device__ __forceinline__ double square_sum(const T* __restrict__ x, int64_t n) {
  constexpr int N = Values<T>::N, U = 4;
  const int64_t packs = n / N;
  double acc[U] = {};
  for (int64_t at = threadIdx.x; at < packs; at += 256 * U) {
    u32x4 r[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      r[u] = u32x4{0, 0, 0, 0};
      if (at + 256 * u < packs) r[u] = load_once(reinterpret_cast<const u32x4_any*>(x + (at + 256 * u) * N));
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int q = 0; q < N; ++q) {
        const double v = Values<T>::get(r[u], q);
        acc[u] = fma(v, v, acc[u]);
      }
    }
  }
  if (threadIdx.x < n - packs * N) {
    const double v = load_as<T>(x + packs * N + threadIdx.x);
    acc[0] = fma(v, v, acc[0]);
  }
  return (acc[0] + acc[1]) + (acc[2] + acc[3]);
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

// Reads each gradient once and adds up squares in fp64: those of fp32 values are exact there, and nothing overflows
// or is lost. The loads bound it: 0.29 G fp32 values in a model's 266 tensors take 178 us with the last
// sum (6.6 TB/s; a streaming read reaches 7.0), and 195 in launches of 64 tensors.
__global__ __launch_bounds__(256) void fl_square_sum_kernel(const NormTable t, int chunk, double* __restrict__ part) {
  __shared__ double s_sum[4];
  const int i = uniform(tensor_of(t, (int)blockIdx.x));
  const int64_t lo = (int64_t)((int)blockIdx.x - t.first[i]) * chunk, left = t.numel[i] - lo;
  const int64_t n = left < chunk ? left : chunk;
  const double v = t.is_bf16[i >> 5] >> (i & 31) & 1 ? square_sum(static_cast<const bf16_bits*>(t.x[i]) + lo, n)
                                : square_sum(static_cast<const float*>(t.x[i]) + lo, n);
  const double sum = block_sum(v, s_sum);
  if (threadIdx.x == 0) part[blockIdx.x] = sum;
}

// out[0] = the norm; out[1] = min(1, max_norm / (norm + 1e-6)), NaN for a norm that is not finite
__global__ __launch_bounds__(1024) void fl_norm_finish_kernel(const double* __restrict__ part, int64_t n,
                                                              float max_norm, float* __restrict__ out, int scaled) {
  __shared__ double s_sum[16];
  double acc = 0.0;
#pragma unroll 4
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
__global__ __launch_bounds__(512) void fl_adamw_factors_kernel(const StepTable t, double lr, const float* lr_ptr,
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

// One value: m and v in, m, v and its root out; the new parameter. The quotient of the update is a product with
// v_rcp_f32 (an ulp; a correctly rounded division is ten operations more and the bf16 8-bit step 8 % slower): the
// update is small beside p. Roots are correctly rounded, the 8-bit codes go by them.
__device__ __forceinline__ float adamw_value(float p, float g, float& m, float& v, float& root, const Factors& f) {
  g = g * f.gs;
  m = m * f.b1 + g * f.b1c;
  v = v * f.b2 + (g * f.b2c) * g;
  root = sqrtf(v);
  return p * f.decay - f.step * (m * __builtin_amdgcn_rcpf(root * f.root_scale + f.eps));
}

template <typename T>
__device__ __forceinline__ u32x4 pack_values(const float* v);
template <>
__device__ __forceinline__ u32x4 pack_values<float>(const float* v) {
  return u32x4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
}
template <>
__device__ __forceinline__ u32x4 pack_values<bf16_bits>(const float* v) {
  return u32x4{bf16_pair(v[0], v[1]), bf16_pair(v[2], v[3]), bf16_pair(v[4], v[5]), bf16_pair(v[6], v[7])};
}

// 16 bytes of parameters and gradients to a thread and turn, and their moments. Bound by the memory, 28 bytes an fp32
// value: 0.29 G values take 1,415 us (5.7 TB/s; four streams read and three written without arithmetic reach 6.1).
template <typename T>
__global__ __launch_bounds__(256) void fl_adamw_kernel(const AdamTable<false> t, const f32x4* __restrict__ hyper,
                                                       float b1, float b1c, float b2, float b2c, float eps) {
  constexpr int N = Values<T>::N;
  const int i = uniform(tensor_of(t, (int)blockIdx.x));
  const f32x4 h = hyper[i];
  if (h[3] != h[3]) return;
  const Factors f = {h[0], h[1], h[2], h[3], b1, b1c, b2, b2c, eps};
  const int64_t lo = (int64_t)((int)blockIdx.x - t.first[i]) * kChunk, left = t.numel[i] - lo;
  const int n = left < kChunk ? (int)left : kChunk, packs = n / N;
  T* p = static_cast<T*>(t.p[i]) + lo;
  const T* g = static_cast<const T*>(t.g[i]) + lo;
  float *ms = static_cast<float*>(t.m[i]) + lo, *vs = static_cast<float*>(t.v[i]) + lo;
#pragma unroll
  for (int u = 0; u < kChunk / N / 256; ++u) {
    const int at = u * 256 + (int)threadIdx.x;
    if (at < packs) {
      const u32x4 pr = load_once(reinterpret_cast<const u32x4_any*>(p + at * N));
      const u32x4 gr = load_once(reinterpret_cast<const u32x4_any*>(g + at * N));
      u32x4 mr[N / 4], vr[N / 4];
#pragma unroll
      for (int w = 0; w < N / 4; ++w) {
        mr[w] = load_once(reinterpret_cast<const u32x4_any*>(ms + at * N + 4 * w));
        vr[w] = load_once(reinterpret_cast<const u32x4_any*>(vs + at * N + 4 * w));
      }
      float o[N];
#pragma unroll
      for (int q = 0; q < N; ++q) {
        float m = __uint_as_float(mr[q / 4][q % 4]), v = __uint_as_float(vr[q / 4][q % 4]), root;
        o[q] = adamw_value(Values<T>::get(pr, q), Values<T>::get(gr, q), m, v, root, f);
        mr[q / 4][q % 4] = __float_as_uint(m);
        vr[q / 4][q % 4] = __float_as_uint(v);
      }
      store_once(reinterpret_cast<u32x4_any*>(p + at * N), pack_values<T>(o));
#pragma unroll
      for (int w = 0; w < N / 4; ++w) {
        store_once(reinterpret_cast<u32x4_any*>(ms + at * N + 4 * w), mr[w]);
        store_once(reinterpret_cast<u32x4_any*>(vs + at * N + 4 * w), vr[w]);
      }
    }
  }
  const int k = packs * N + (int)threadIdx.x;
  if (k < n) {
    float m = ms[k], v = vs[k], root;
    store_as(p + k, adamw_value(load_as<T>(p + k), load_as<T>(g + k), m, v, root, f));
    ms[k] = m;
    vs[k] = v;
  }
}

__device__ __forceinline__ float code_value(uint32_t codes, int q) {  // (q a constant once unrolled)
  return q == 0   ? __builtin_amdgcn_cvt_f32_fp8((int)codes, 0)
         : q == 1 ? __builtin_amdgcn_cvt_f32_fp8((int)codes, 1)
         : q == 2 ? __builtin_amdgcn_cvt_f32_fp8((int)codes, 2)
                  : __builtin_amdgcn_cvt_f32_fp8((int)codes, 3);
}

__device__ __forceinline__ uint32_t four_codes(const float* y) {
  const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], lo, true);
}

// value q of a pack, to be written
__device__ __forceinline__ void set_value(u32x4& r, int q, float v) { r[q] = __float_as_uint(v); }
__device__ __forceinline__ void set_value(u32x4& r, int q, bf16_bits v) {
  r[q >> 1] = q & 1 ? (r[q >> 1] & 0xffffu) | (uint32_t)v << 16 : (r[q >> 1] & 0xffff0000u) | v;
}

// N codes, of 4 or 8 bytes
template <int N>
struct Codes;
template <>
struct Codes<4> {
  uint32_t w[1] = {0};
  __device__ __forceinline__ void load(const uint8_t* p) { w[0] = load_once(reinterpret_cast<const u32_any*>(p)); }
  __device__ __forceinline__ void store(uint8_t* p) const { store_once(reinterpret_cast<u32_any*>(p), w[0]); }
};
template <>
struct Codes<8> {
  uint32_t w[2] = {0, 0};
  __device__ __forceinline__ void load(const uint8_t* p) {
    const u32x2 v = load_once(reinterpret_cast<const u32x2_any*>(p));
    w[0] = v.x;
    w[1] = v.y;
  }
  __device__ __forceinline__ void store(uint8_t* p) const {
    store_once(reinterpret_cast<u32x2_any*>(p), u32x2{w[0], w[1]});
  }
};

// largest of 64 or of each half's 32 lanes
template <int LANES>
__device__ __forceinline__ float lanes_max(float v) {
  if constexpr (LANES == 64) return wave_max(v);
  v = dpp_max<0xb1>(v);
  v = dpp_max<0x4e>(v);
  v = dpp_max<0x141>(v);
  v = dpp_max<0x140>(v);
  const u32x2 a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(a.x), __uint_as_float(a.y));
}

// A block of 256 values to a wave (fp32) or to half of one (bf16), 16 bytes of them to a lane, 2,048 values to four
// waves with all their loads ahead of the maths. m is held as the e4m3 code of m (448 / max|m|), v as that of its
// root r (448 / max r), with max / 448 beside: a root keeps v's range in half the octaves, and one that is not 0 keeps
// at least the smallest code, since a v that rounds to 0 under an m that does not would let the next step with a small
// gradient run away. Bound by the memory, 16 bytes an fp32 value: 0.29 G values take 770 us (6.1 TB/s).
template <typename T>
__global__ __launch_bounds__(256) void fl_adamw8_kernel(const AdamTable<true> t, const f32x4* __restrict__ hyper,
                                                        float b1, float b1c, float b2, float b2c, float eps) {
  constexpr int N = Values<T>::N, LANES = kBlock / N, GROUPS = 64 / LANES, U = kChunk / kBlock / 4 / GROUPS;
  const int i = uniform(tensor_of(t, (int)blockIdx.x));
  const f32x4 h = hyper[i];
  if (h[3] != h[3]) return;
  const Factors f = {h[0], h[1], h[2], h[3], b1, b1c, b2, b2c, eps};
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int64_t lo = (int64_t)((int)blockIdx.x - t.first[i]) * kChunk, left = t.numel[i] - lo;
  const int n = left < kChunk ? (int)left : kChunk;
  T* p = static_cast<T*>(t.p[i]) + lo;
  const T* g = static_cast<const T*>(t.g[i]) + lo;
  uint8_t *mc = static_cast<uint8_t*>(t.m[i]) + lo, *vc = static_cast<uint8_t*>(t.v[i]) + lo;
  float *ms = t.ms[i] + lo / kBlock, *vs = t.vs[i] + lo / kBlock;
  u32x4 pr[U] = {}, gr[U] = {};
  Codes<N> mr[U], vr[U];
  float sm[U] = {}, sv[U] = {};
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int b = (u * 4 + wave) * GROUPS + lane / LANES, k = b * kBlock + lane % LANES * N;
    if (b * kBlock < n) {
      sm[u] = ms[b];
      sv[u] = vs[b];
    }
    if (k + N <= n) {
      pr[u] = load_once(reinterpret_cast<const u32x4_any*>(p + k));
      gr[u] = load_once(reinterpret_cast<const u32x4_any*>(g + k));
      mr[u].load(mc + k);
      vr[u].load(vc + k);
    } else if (k < n) {
#pragma unroll
      for (int q = 0; q < N - 1; ++q) {
        if (k + q < n) {
          set_value(pr[u], q, p[k + q]);
          set_value(gr[u], q, g[k + q]);
          mr[u].w[q / 4] |= (uint32_t)mc[k + q] << (8 * (q % 4));
          vr[u].w[q / 4] |= (uint32_t)vc[k + q] << (8 * (q % 4));
        }
      }
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int b = (u * 4 + wave) * GROUPS + lane / LANES, k = b * kBlock + lane % LANES * N;
    if ((u * 4 + wave) * GROUPS * kBlock >= n) break;  // (wave-uniform)
    float o[N], m[N], r[N], top_m = 0.f, top_r = 0.f;
#pragma unroll
    for (int q = 0; q < N; ++q) {  // (behind the tensor's end all is 0 and stays 0)
      m[q] = code_value(mr[u].w[q / 4], q % 4) * sm[u];
      const float root = code_value(vr[u].w[q / 4], q % 4) * sv[u];
      float v = root * root;
      o[q] = adamw_value(Values<T>::get(pr[u], q), Values<T>::get(gr[u], q), m[q], v, r[q], f);
      top_m = fmaxf(top_m, fabsf(m[q]));
      top_r = fmaxf(top_r, r[q]);
    }
    top_m = lanes_max<LANES>(top_m);
    top_r = lanes_max<LANES>(top_r);
    const float inv_m = top_m >= kTiny ? 1.0f / top_m * kTopCode : 0.f;
    const float inv_r = top_r >= kTiny ? 1.0f / top_r * kTopCode : 0.f;
    Codes<N> mo, vo;
#pragma unroll
    for (int q = 0; q < N; ++q) {
      m[q] *= inv_m;
      r[q] *= inv_r;
      if (r[q] > 0.f && r[q] < kSmallest) r[q] = kSmallest;
    }
#pragma unroll
    for (int w = 0; w < N / 4; ++w) {
      mo.w[w] = four_codes(m + 4 * w);
      vo.w[w] = four_codes(r + 4 * w);
    }
    if (k + N <= n) {
      store_once(reinterpret_cast<u32x4_any*>(p + k), pack_values<T>(o));
      mo.store(mc + k);
      vo.store(vc + k);
    } else if (k < n) {
#pragma unroll
      for (int q = 0; q < N - 1; ++q) {
        if (k + q < n) {
          store_as(p + k + q, o[q]);
          mc[k + q] = (uint8_t)(mo.w[q / 4] >> (8 * (q % 4)));
          vc[k + q] = (uint8_t)(vo.w[q / 4] >> (8 * (q % 4)));
        }
      }
    }
    if (lane % LANES == 0 && b * kBlock < n) {
      ms[b] = top_m >= kTiny ? top_m * (1.0f / kTopCode) : 0.f;
      vs[b] = top_r >= kTiny ? top_r * (1.0f / kTopCode) : 0.f;
    }
  }
}

constexpr int64_t kMaxNumel = (int64_t)1 << 34;  // 2^23 blocks: a tensor always fits a launch
constexpr int64_t kMaxTensors = 1 << 20;

// Fills `table` with tensors from `i` on, empty ones too; returns the index after the last one taken.
template <typename Table, typename Put>
int64_t fill_table(Table& table, int64_t n, const int64_t* numel, int64_t i, int chunk, Put put) {
  table.n = 0;
  table.first[0] = 0;
  for (; i < n && table.n < Table::kSize; ++i) {
    const int64_t blocks = cdiv(numel[i], chunk);
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
    i = fill_table(t, n, numel, i, kChunk, [&](int k, int64_t j) {
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

// Values of a block of the norm: 4,096 up to 32,768, as many as leave 1,024 blocks (13 M values: 8,192 of them
// 13.5 us, 4,096 of them 14.9; 0.29 G: 16,384 of them 180 us, 32,768 178, 65,536 183, 131,072 201).
int norm_chunk(int64_t n, const int64_t* numel) {
  int64_t total = 0;
  for (int64_t i = 0; i < n; ++i) total += numel[i];
  int chunk = 4096;
  while (chunk < 32768 && total / chunk > 2048) chunk *= 2;
  return chunk;
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
  const int chunk = norm_chunk(n, numel);
  for (int64_t i = 0; i < n; ++i) blocks += cdiv(numel[i], chunk);
  return (size_t)(blocks > 0 ? blocks : 1) * sizeof(double);
}

int fl_grad_norm(int64_t n, const void* const* grads, const int* dtypes, const int64_t* numel, float max_norm,
                 int scaled, float* out, void* workspace, size_t workspace_bytes, void* stream) {
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
  const int chunk = norm_chunk(n, numel);
  for (int64_t i = 0; i < n;) {
    NormTable t = {};
    i = fill_table(t, n, numel, i, chunk, [&](int k, int64_t j) {
      t.x[k] = grads[j];
      t.is_bf16[k >> 5] |= (uint32_t)(dtypes[j] == FL_DTYPE_BF16) << (k & 31);
    });
    const int blocks = t.first[t.n];
    if (blocks == 0) continue;
    fl_square_sum_kernel<<<(unsigned)blocks, 256, 0, s>>>(t, chunk, part + done);
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
                  const int64_t* numel, int64_t* const* steps, double lr, const float* lr_ptr, double beta1,
                  double beta2, double eps, double weight_decay, const float* grad_scale, void* workspace,
                  size_t workspace_bytes, void* stream) {
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
    fl_adamw_factors_kernel<<<1, cdiv(t.n, 64) * 64, 0, s>>>(t, lr, lr_ptr, beta1, beta2, weight_decay, grad_scale,
                                                             hyper + i);
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
