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
constexpr float kMinTemperature = 9.5367431640625e-7f, kMaxTemperature = 1048576.0f;  // 2^-20, 2^20
constexpr float kLn2 = 0.6931471805599453f;

struct Rows {
  int64_t inner;                      // row r is (r / inner, r % inner)
  int64_t stride_outer, stride_inner; // of the logits, in elements
  int64_t token_outer, token_inner;   // of the tokens
  // where row r is; most callers have one group of rows, and a 64-bit division is 200 instructions ahead of the
  // loads
  __device__ __forceinline__ void find(int64_t r, int64_t& logit_at, int64_t& token_at) const {
    const bool wide = (uint64_t)r >> 32 || (uint64_t)inner >> 32;
    const int64_t o = r < inner ? 0 : wide ? r / inner : (uint32_t)r / (uint32_t)inner;
    const int64_t i = r - o * inner;
    logit_at = o * stride_outer + i * stride_inner;
    token_at = o * token_outer + i * token_inner;
  }
};

// Order of the alternatives as an integer: larger values first, -0 as 0, NaN above all, then the lower index.
// Every key lies strictly between 0 and ~0, which stand for none and for no limit.
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);
  return x != x ? 0xfffffffeu : b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ uint64_t rank_key(float x, uint32_t index) {
  return (uint64_t)order_of(x) << 32 | (0xffffffffu - index);
}

__device__ __forceinline__ float key_value(uint64_t key) {
  const uint32_t b = (uint32_t)(key >> 32);
  return b == 0xfffffffeu ? __uint_as_float(0x7fc00000u) : __uint_as_float(b & 0x80000000u ? b ^ 0x80000000u : ~b);
}

__device__ __forceinline__ float quiet_nan() { return __uint_as_float(0x7fc00000u); }

template <typename T>
struct Pack;
template <>
struct Pack<bf16_bits> {
  static constexpr int N = 8;
  static constexpr uint32_t kNone = 0xff80ff80u;  // -inf
  __device__ __forceinline__ static float get(const u32x4& v, int q) {
    return q & 1 ? bf16_hi(v[q >> 1]) : bf16_lo(v[q >> 1]);
  }
};
template <>
struct Pack<float> {
  static constexpr int N = 4;
  static constexpr uint32_t kNone = 0xff800000u;
  __device__ __forceinline__ static float get(const u32x4& v, int q) { return __uint_as_float(v[q]); }
};

template <int CTRL>
__device__ __forceinline__ uint64_t dpp_key_max(uint64_t v) {
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(v >> 32), CTRL, 0xf, 0xf, true);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
  const uint64_t o = (uint64_t)hi << 32 | lo;
  return o > v ? o : v;
}
// largest key of the wave, in every lane (the steps of wave_max)
__device__ __forceinline__ uint64_t key_max(uint64_t v) {
  v = dpp_key_max<0xb1>(v);
  v = dpp_key_max<0x4e>(v);
  v = dpp_key_max<0x141>(v);
  v = dpp_key_max<0x140>(v);
  u32x2 h = __builtin_amdgcn_permlane16_swap((uint32_t)(v >> 32), (uint32_t)(v >> 32), false, false);
  u32x2 l = __builtin_amdgcn_permlane16_swap((uint32_t)v, (uint32_t)v, false, false);
  uint64_t a = (uint64_t)h.x << 32 | l.x, b = (uint64_t)h.y << 32 | l.y;
  v = a > b ? a : b;
  h = __builtin_amdgcn_permlane32_swap((uint32_t)(v >> 32), (uint32_t)(v >> 32), false, false);
  l = __builtin_amdgcn_permlane32_swap((uint32_t)v, (uint32_t)v, false, false);
  a = (uint64_t)h.x << 32 | l.x;
  b = (uint64_t)h.y << 32 | l.y;
  return a > b ? a : b;
}

constexpr int kCand = 512;    // candidates for the alternatives that a block ranks
// Alternatives up to which 64 groups bound them, all 256 threads' maxima above: fewer ballots against more
// candidates (of normal logits about 25 for 20, 45 for 32, 65 for 40, 300 for 64). 8,188 rows of 16,384 bf16 with
// entropy take 55 us with 5 and 60 by 256 groups, 61 and 64 with 20, 66 and 67 with 32, 70 and 69 with 40, 75 and 71
// with 48, 378 and 77 with 64; 999 rows of 32,001 fp32 and 64 of 16,384 cross between 32 and 40 as well.
constexpr int kFewTop = 32;
constexpr float kPlainScale = 1048576.0f;  // below this |m| c, x c - fl(m c) is as good as (x - m) c

// What a row's results are made of: m, log2 of s, the mean of d log2(e) under the distribution.
struct RowStats {
  float m, log2_s, mean;
  bool empty;
  float inv_t;
  // from the sum: a row of -inf alone adds up to 0; one with NaN or +inf to NaN, which the maximum may have missed
  __device__ __forceinline__ void settle(float sum) {
    empty = sum == 0.f;
    if (sum != sum) m = sum;
    log2_s = __builtin_amdgcn_logf(sum);
  }
  __device__ __forceinline__ float log_sum() const { return log2_s * kLn2; }
  // (a product with the rounded 1 / T: up to 2^-24 |d| more than a quotient is off by, as every d of the sum has)
  __device__ __forceinline__ float logprob(float x) const {
    return empty ? -INFINITY : (x - m) * inv_t - log2_s * kLn2;
  }
  __device__ __forceinline__ float entropy() const { return empty ? 0.f : (log2_s - mean) * kLn2; }
};

struct Outputs {
  const int64_t* tokens;
  int64_t ignore;
  int K;
  float* logprobs;
  float* entropy;
  float* top_lp;
  int64_t* top_tok;
  float* stats;
};

__device__ __forceinline__ void write_row(const Outputs& out, int64_t row, const RowStats& st, int64_t t, int V,
                                          float xt) {
  out.logprobs[row] = t == out.ignore ? 0.f : t >= 0 && t < V ? st.logprob(xt) : quiet_nan();
  if (out.entropy) out.entropy[row] = st.entropy();
  if (out.stats) {
    out.stats[2 * row] = st.m;
    out.stats[2 * row + 1] = st.log_sum();
  }
}

// One block to a row, or to a segment of one (gridDim.y of them): its logits stay in registers, NV packs of 16 bytes
// to a thread, for the maximum, the sums and the alternatives, so that memory is read once. With the segment's maximum
// known, e^d is one fused product and one power (x c - m c, c = log2(e) / T; the rounding error of m c is put back
// into the log at the end), and no sum is ever rescaled. The memory bounds it where rows are many: 8,192 rows of
// 16,384 bf16 take 42 us (6.4 TB/s; a streaming read reaches 7.0), 29 of which their vector instructions fill too (5.5
// a logit, 7.5 with entropy, of four cycles each and eight for the power). With entropy and 20 alternatives they take
// 61, of which the instructions fill 48 and the memory 39. One row of 131,072 is two launches and 12 us.
//
// Alternatives: the threads' maxima (in 64 groups where K is small) give a value that at least K logits reach: their
// K-th largest, to 16 bits. Only logits from there up are candidates, little more than K of them in text; they are
// ranked by counting. Rows that hold NaN or +inf, and rows with more candidates than fit (equal logits), are
// searched by halving instead: for the K-th largest value, then for the index up to which those equal to it count.
template <typename T, int THREADS, int NV, bool ENT, bool TOP>
__global__ __launch_bounds__(THREADS) void fl_token_logprobs_kernel(
    const T* __restrict__ logits, Rows rows, int64_t n_rows, int V, int seg_len, float inv_t, Outputs out,
    f32x4* __restrict__ part, uint64_t* __restrict__ part_keys) {
  constexpr int N = Pack<T>::N, WAVES = THREADS / 64;
  __shared__ float s_max[THREADS], s_sum[2 * WAVES];
  __shared__ unsigned long long s_cand[kCand];
  __shared__ int s_n, s_count[WAVES];
  const int K = TOP ? out.K : 0;
  const int lo = (int)blockIdx.y * seg_len, len = V - lo < seg_len ? V - lo : seg_len;
  const bool whole = gridDim.y == 1;
  const float c = inv_t * kLog2e;
  for (int64_t row = blockIdx.x; row < n_rows; row += gridDim.x) {
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));  // (what depends on it is computed where it is wanted, not kept over the rows)
    const int lane = tid & 63, wave = uniform(tid >> 6);
    int64_t logit_at, token_at;
    rows.find(row, logit_at, token_at);
    const int64_t t = out.tokens[token_at];
    if (!TOP && !ENT && t == out.ignore) {  // nothing of this row is asked for
      if (whole && tid == 0) {
        out.logprobs[row] = 0.f;
        if (out.stats) out.stats[2 * row] = out.stats[2 * row + 1] = 0.f;
      }
      continue;
    }
    const T* row_x = logits + logit_at;
    const T* x = row_x + lo;
    // packs from the first 16-byte border on (8,192 rows of 16,383 bf16 logits: 43 us, and 58 from the row's start)
    const int ahead = (int)(-(uintptr_t)x % 16 / sizeof(T)), head = ahead < len ? ahead : len;
    const int packs = (len - head) / N, tail = head + packs * N;
    float xt = 0.f;
    if (whole && tid == 0 && t >= 0 && t < V) xt = load_as<T>(row_x + t);
    u32x4 v[NV];
    const auto load = [&](auto get) {
      // (a uniform address and 32 bits beside: no address of its own to a lane and pack)
      const auto place = [&](int i) {
        const char* from = reinterpret_cast<const char*>(x + head + i * THREADS * N);
        return reinterpret_cast<const u32x4*>(from + (uint32_t)tid * 16u);
      };
      if (packs == NV * THREADS) {  // all of the tile: nothing to stand in for
#pragma unroll
        for (int i = 0; i < NV; ++i) v[i] = get(place(i));
        return;
      }
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int j = i * THREADS + tid;
        v[i] = u32x4{Pack<T>::kNone, Pack<T>::kNone, Pack<T>::kNone, Pack<T>::kNone};
        if (j < packs) v[i] = get(place(i));
      }
    };
    // Logits that no backward will read again pass the caches by (8,192 rows of 16,384 bf16: 42 us, and 48 through
    // them; where one follows the pair with entropy takes 141 us so, and 133 through them).
    if (out.stats) load([](const u32x4* p) { return *p; });
    else load([](const u32x4* p) { return __builtin_nontemporal_load(p); });
    // the logits ahead of the first pack and behind the last, one to a thread (fewer than 8 each), len for none
    const auto rest_place = [&](int t) { return t < head ? t : t >= 8 && t - 8 < len - tail ? tail + t - 8 : len; };
    float rest = -INFINITY;
    if (rest_place(tid) < len) rest = load_as<T>(x + rest_place(tid));
    // f(logit, i, q) of all the thread's logits, and of -inf for those it lacks
    const auto each = [&](auto f) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          // (opaque, or the compiler keeps what one pass unpacked for the next: twice the registers)
          asm volatile("" : "+v"(v[i][w]));
#pragma unroll
          for (int q = w * N / 4; q < (w + 1) * N / 4; ++q) f(Pack<T>::get(v[i], q), i, q);
        }
      }
      f(rest, NV, 0);
    };
    // f(logit, place in the segment), places that it lacks from len up
    const auto for_places = [&](auto f) {
      for (int j = tid; __ballot(j < packs); j += THREADS) {
        u32x4 again = {Pack<T>::kNone, Pack<T>::kNone, Pack<T>::kNone, Pack<T>::kNone};
        if (j < packs) again = *reinterpret_cast<const u32x4*>(x + head + j * N);
#pragma unroll
        for (int q = 0; q < N; ++q) f(Pack<T>::get(again, q), j < packs ? head + j * N + q : len);
      }
      f(rest, rest_place(tid));
    };
    if (TOP && tid == 0) s_n = 0;
    float mine = rest, pack_top[TOP ? NV : 1];
    if constexpr (TOP) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        pack_top[i] = Pack<T>::get(v[i], 0);
#pragma unroll
        for (int q = 1; q < N; ++q) pack_top[i] = fmaxf(pack_top[i], Pack<T>::get(v[i], q));
        mine = fmaxf(mine, pack_top[i]);
      }
    } else {
      each([&](float a, int, int) { mine = fmaxf(mine, a); });
    }
    s_max[tid] = mine;
    __syncthreads();
    float group = s_max[lane];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) group = fmaxf(group, s_max[w * 64 + lane]);
    RowStats st;
    st.inv_t = inv_t;
    st.m = wave_max(group);
    const float base = st.m == -INFINITY ? 0.f : st.m, shift = base * c;
    float sum = 0.f, ent = 0.f, resid = 0.f;
    const auto add = [&](float d) {
      const float e = __builtin_amdgcn_exp2f(d);
      sum += e;
      if constexpr (ENT) ent = fmaf(e, fmaxf(d, -1000.f), ent);  // (0 times -inf is no number)
    };
    if (__builtin_fabsf(shift) < kPlainScale) {
      resid = fmaf(base, c, -shift);
      each([&](float a, int, int) { add(fmaf(a, c, -shift)); });
    } else {
      each([&](float a, int, int) { add((a - base) * c); });
    }
    sum = wave_sum(sum);
    if constexpr (ENT) ent = wave_sum(ent);
    if constexpr (WAVES > 1) {
      if (lane == 0) {
        s_sum[wave] = sum;
        if constexpr (ENT) s_sum[WAVES + wave] = ent;
      }
      __syncthreads();
      sum = s_sum[0];
      if constexpr (ENT) ent = s_sum[WAVES];
#pragma unroll
      for (int w = 1; w < WAVES; ++w) {
        sum += s_sum[w];
        if constexpr (ENT) ent += s_sum[WAVES + w];
      }
    }
    st.settle(sum);
    st.log2_s -= resid;
    st.mean = ENT ? ent / sum - resid : 0.f;
    if (tid == 0) {
      if (whole) write_row(out, row, st, t, V, xt);
      else part[row * gridDim.y + blockIdx.y] = f32x4{st.m, st.log2_s, st.mean, 0.f};
    }
    if constexpr (TOP) {
      const auto put = [&](int k, uint64_t key) {
        if (whole) {
          out.top_tok[row * K + k] = 0xffffffffu - (uint32_t)key;
          out.top_lp[row * K + k] = st.logprob(key_value(key));
        } else {
          part_keys[(row * gridDim.y + blockIdx.y) * K + k] = key;
        }
      };
      const auto push = [&](float a, int at) {  // at: where in the segment
        const int k = atomicAdd(&s_n, 1);
        if (k < kCand) s_cand[k] = (uint64_t)__float_as_uint(a) << 32 | (uint32_t)at;
      };
      int n = kCand + 1;
      uint32_t bound = 0;  // the upper half of order_of of a value that K logits reach
      if (sum == sum) {
        if (WAVES > 1 && K > kFewTop) {
          uint32_t g[WAVES];
#pragma unroll
          for (int w = 0; w < WAVES; ++w) g[w] = order_of(s_max[w * 64 + lane]) >> 16;
          for (int bit = 15; bit >= 0; --bit) {
            const uint32_t test = bound | 1u << bit;
            int reach = 0;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) reach += __popcll(__ballot(g[w] >= test));
            if (reach >= K) bound = test;
          }
        } else {
          const uint32_t g = order_of(group) >> 16;
#pragma unroll
          for (int bit = 15; bit >= 0; --bit) {
            const uint32_t test = bound | 1u << bit;
            if (__popcll(__ballot(g >= test)) >= K) bound = test;
          }
        }
        // The packs that hold a candidate are read once more.
        const auto scan = [&](auto in_pack, auto is) {
          uint32_t hit = 0;
#pragma unroll
          for (int i = 0; i < NV; ++i) hit |= in_pack(i) ? 1u << i : 0u;
          while (hit) {
            const int at = head + (__builtin_ctz(hit) * THREADS + tid) * N;
            hit &= hit - 1;
            const u32x4 again = *reinterpret_cast<const u32x4*>(x + at);
#pragma unroll
            for (int q = 0; q < N; ++q) {
              const float a = Pack<T>::get(again, q);
              if (is(a, at + q)) push(a, at + q);
            }
          }
        };
        if (bound > 0x007fu) {
          const float least = __uint_as_float(bound & 0x8000u ? bound << 16 ^ 0x80000000u : ~(bound << 16));
          scan([&](int i) { return pack_top[i] >= least; }, [&](float a, int) { return a >= least; });
          if (rest >= least) push(rest, rest_place(tid));
        } else {
          // fewer than K groups hold a logit above -inf: all of those, and the masked ones of lowest index
          scan([&](int i) {
                 const int j = i * THREADS + tid;
                 return j < packs && (pack_top[i] > -INFINITY || head + j * N < 2 * K);
               },
               [&](float a, int at) { return a > -INFINITY || at < 2 * K; });
          const int at = rest_place(tid);
          if (at < len && (rest > -INFINITY || at < 2 * K)) push(rest, at);
        }
        __syncthreads();
        n = s_n;
      }
      if (n > kCand) {  // (block-uniform)
        const int want = K < len ? K : len;
        // how many of the segment's logits fulfil is(order, place), over the block
        const auto count = [&](auto is) {
          int mine_n = 0;
          for_places([&](float a, int at) { mine_n += __popcll(__ballot(at < len && is(order_of(a), at))); });
          __syncthreads();
          if (lane == 0) s_count[wave] = mine_n;
          __syncthreads();
          int all = s_count[0];
#pragma unroll
          for (int w = 1; w < WAVES; ++w) all += s_count[w];
          return all;
        };
        uint32_t low = sum == sum ? bound << 16 : 0, high = sum == sum ? order_of(base) : 0xffffffffu;
        while (low < high) {
          const uint32_t mid = low + (high - low) / 2 + 1;
          if (count([&](uint32_t o, int) { return o >= mid; }) >= want) low = mid;
          else high = mid - 1;
        }
        const int need = want - count([&](uint32_t o, int) { return o > low; });
        int last = len - 1;
        for (int from = 0; from < last;) {
          const int mid = (from + last) / 2;
          if (count([&](uint32_t o, int at) { return o == low && at <= mid; }) >= need) last = mid;
          else from = mid + 1;
        }
        __syncthreads();
        if (tid == 0) s_n = 0;
        __syncthreads();
        for_places([&](float a, int at) {
          const uint32_t o = order_of(a);
          if (at < len && (o > low || (o == low && at <= last))) push(a, at);
        });
        __syncthreads();
        n = s_n;
      }
      const auto key_at = [&](int i) {
        const uint64_t c = s_cand[i];
        return rank_key(__uint_as_float((uint32_t)(c >> 32)), (uint32_t)lo + (uint32_t)c);
      };
      if (n <= 64) {  // one wave, a candidate to a lane
        if (wave == 0) {
          const uint64_t key = lane < n ? key_at(lane) : 0;
          int rank = 0;
          // (keys broadcast by the LDS: half the vector instructions of reading them from lanes, 61.6 us against 63.3
          // for 8,188 rows of 16,384 bf16 with entropy and 20 alternatives)
          s_cand[lane] = key;
          __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll 4
          for (int j = 0; j < n; ++j) rank += s_cand[j] > key;
          if (lane < n && rank < K) put(rank, key);
        }
      } else {
        for (int i = tid; i < n; i += THREADS) s_cand[i] = key_at(i);
        __syncthreads();
        for (int i = tid; i < n; i += THREADS) {
          const uint64_t key = s_cand[i];
          int rank = 0;
#pragma unroll 4
          for (int j = 0; j < n; ++j) rank += s_cand[j] > key;
          if (rank < K) put(rank, key);
        }
      }
      for (int k = n + tid; k < K; k += THREADS) put(k, 0);  // (a segment of fewer than K)
    }
    __syncthreads();  // the next row takes the shared memory
  }
}

// Joins a row's segments, one thread to a segment: their sums relative to the row's maximum, and their sorted lists of
// alternatives. SMALL, up to 64 segments: the K-th largest of the lists' first K / segments + 1 keys is a key that K
// reach; those that do, little more than K, are ranked by counting. Where they are more than fit, and for up to 1,024
// segments, K times the largest of the lists' heads is taken. (A row of 131,072 fp32, both launches: with 20
// alternatives 12.4 us, with 64 17.3; by heads alone 14.2 and 27.8.)
template <typename T, int THREADS, bool SMALL>
__global__ __launch_bounds__(THREADS) void fl_token_logprobs_join_kernel(
    const T* __restrict__ logits, Rows rows, int64_t n_rows, int V, int segments, float inv_t, Outputs out,
    const f32x4* __restrict__ part, const uint64_t* __restrict__ part_keys) {
  constexpr int WAVES = THREADS / 64;
  __shared__ float s_f[3 * WAVES];
  __shared__ unsigned long long s_best[2][WAVES], s_keys[SMALL ? 64 * kMaxTop : 1], s_cand[SMALL ? kCand : 1], s_bound;
  __shared__ int s_n;
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), K = out.K;
  const float c = inv_t * kLog2e;
  for (int64_t row = blockIdx.x; row < n_rows; row += gridDim.x) {
    int64_t logit_at, token_at;
    rows.find(row, logit_at, token_at);
    const int64_t t = out.tokens[token_at];
    float xt = 0.f;
    if (tid == 0 && t >= 0 && t < V) xt = load_as<T>(logits + logit_at + t);
    f32x4 p = {-INFINITY, -INFINITY, 0.f, 0.f};
    if (tid < segments && !(t == out.ignore && K == 0 && !out.entropy)) p = part[row * segments + tid];
    const uint64_t* keys = part_keys + row * segments * K;
    if constexpr (SMALL) {
#pragma unroll 2
      for (int i = tid; i < segments * K; i += THREADS) s_keys[i] = keys[i];
      if (tid == 0) {
        s_n = 0;
        s_bound = 1;  // (no list's filling of 0)
      }
    }
    RowStats st;
    st.inv_t = inv_t;
    st.m = wave_max(p[0]);
    if (lane == 0) s_f[wave] = st.m;
    __syncthreads();
    for (int w = 0; w < WAVES; ++w) st.m = fmaxf(st.m, s_f[w]);
    // d log2(e) of the segment's own maximum; a segment of -inf alone adds nothing
    const float d = (p[0] - st.m) * c;
    const bool live = p[0] != -INFINITY;
    const float s = live ? __builtin_amdgcn_exp2f(d + p[1]) : 0.f;
    float sum = wave_sum(s), ent = wave_sum(live && s != 0.f ? s * (p[2] + d) : 0.f);
    if (lane == 0) {
      s_f[WAVES + wave] = sum;
      s_f[2 * WAVES + wave] = ent;
    }
    __syncthreads();
    sum = ent = 0.f;
    for (int w = 0; w < WAVES; ++w) {
      sum += s_f[WAVES + w];
      ent += s_f[2 * WAVES + w];
    }
    st.settle(sum);
    st.mean = ent / sum;
    if (tid == 0) write_row(out, row, st, t, V, xt);
    const auto put = [&](int k, uint64_t key) {
      out.top_tok[row * K + k] = 0xffffffffu - (uint32_t)key;
      out.top_lp[row * K + k] = st.logprob(key_value(key));
    };
    if constexpr (SMALL) {
      if (K == 0) {  // (block-uniform)
        __syncthreads();
        continue;
      }
      const int each = K / segments + 1, some = segments * each;  // K < some <= K + 64, each <= K
      if (tid < some) {
        const uint64_t key = s_keys[tid / each * K + tid % each];
        int rank = 0;
#pragma unroll 4
        for (int j = 0; j < segments; ++j)
          for (int q = 0; q < each; ++q) rank += s_keys[j * K + q] > key;
        if (rank == K - 1 && key) s_bound = key;  // (keys other than 0 are unique)
      }
      __syncthreads();
      const uint64_t bound = s_bound;
      for (int i = tid; i < segments * K; i += THREADS) {
        const uint64_t key = s_keys[i];
        if (key < bound) continue;
        const int at = atomicAdd(&s_n, 1);
        if (at < kCand) s_cand[at] = key;
      }
      __syncthreads();
      const int n = s_n;
      if (n <= kCand) {
        for (int i = tid; i < n; i += THREADS) {
          const uint64_t key = s_cand[i];
          int rank = 0;
#pragma unroll 4
          for (int j = 0; j < n; ++j) rank += s_cand[j] > key;
          if (rank < K) put(rank, key);
        }
        __syncthreads();
        continue;
      }
    }
    const auto key_of = [&](int k) -> uint64_t {
      if (tid >= segments || k >= K) return 0;
      if constexpr (SMALL) return s_keys[tid * K + k];
      else return keys[tid * K + k];
    };
    if (!SMALL || wave == 0) {  // (SMALL: the first wave holds all lists)
      int at = 0;
      uint64_t head = key_of(0);
      for (int k = 0; k < K; ++k) {
        uint64_t best = key_max(head);
        if constexpr (!SMALL) {
          if (lane == 0) s_best[k & 1][wave] = best;
          __syncthreads();
          for (int w = 0; w < WAVES; ++w) best = s_best[k & 1][w] > best ? s_best[k & 1][w] : best;
        }
        if (head == best) head = key_of(++at);
        if (tid == 0) put(k, best);
      }
    }
    __syncthreads();
  }
}

// Gradients: a block writes kBackPacks packs to a thread of one row, then the logits that carry a gradient of their
// own (the given token, the alternatives). With L = m c + log2 s (c = log2(e) / T) split into its
// rounded value and the rest, p = 2^(x c - L) is one fused product and one power, and the row's constants make
//   dx = -(p / T) (g + sum g_k + h (ln p + H))
// two more operations, one without h. A row whose gradients are all 0 gets zeros whatever its logits hold.
// Bound by the memory: 8,192 rows of 16,384 bf16 take 92 us (5.8 TB/s of reads and writes; a streaming copy reaches
// 6.1 with four packs to a thread and 6.7 with one), 999 of 32,001 fp32 with entropy and 8 alternatives 53. 4 packs
// to a thread: with 2 those take 91 and 55 (104 and 115 with 20 alternatives), with 8 93 and 149. At least six waves
// to a SIMD (79 registers): 58 us for the 999 rows at the compiler's own five, and 120 for the 8,192 at eight.
constexpr int kBackPacks = 4;

template <typename T>
__device__ __forceinline__ void store_pack(T* p, const float* v);
template <>
__device__ __forceinline__ void store_pack<bf16_bits>(bf16_bits* p, const float* v) {
  u32x4 w;
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = bf16_pair(v[2 * i], v[2 * i + 1]);
  __builtin_nontemporal_store(w, reinterpret_cast<u32x4*>(p));
}
template <>
__device__ __forceinline__ void store_pack<float>(float* p, const float* v) {
  u32x4 w;
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = __float_as_uint(v[i]);
  __builtin_nontemporal_store(w, reinterpret_cast<u32x4*>(p));
}

template <typename T, int THREADS, bool ENT>
__global__ __launch_bounds__(THREADS, 6) void fl_token_logprobs_backward_kernel(
    const T* __restrict__ logits, Rows rows, int64_t n_rows, int V, const int64_t* __restrict__ tokens,
    int64_t ignore, float inv_t, int K, const float* __restrict__ stats, const float* __restrict__ entropy,
    const int64_t* __restrict__ top_tok, const float* __restrict__ g_lp, const float* __restrict__ g_ent,
    const float* __restrict__ g_top, T* __restrict__ grad) {
  constexpr int N = Pack<T>::N, kChunk = THREADS * kBackPacks * N;
  const int tid = threadIdx.x, lane = tid & 63;
  const float c = inv_t * kLog2e;
  for (int64_t at_row = blockIdx.x; at_row < n_rows; at_row += gridDim.x) {
    const int64_t row = n_rows - 1 - at_row;  // the forward's last rows first: they may still be cached
    int64_t logit_at, token_at;
    rows.find(row, logit_at, token_at);
    const T* x = logits + logit_at;
    T* out = grad + row * V;
    // Chunks from the gradient row's first 128-byte line on, so that no line is written in parts (8,192 rows of 16,383
    // bf16: 93 us, and 120 from the row's start); the logits ahead of it are the first chunk's too.
    const int ahead = (int)(-(uintptr_t)out % 128 / sizeof(T)), first = ahead + (int)blockIdx.y * kChunk;
    const int lo = blockIdx.y ? first : 0, hi = V - first < kChunk ? V : first + kChunk;
    const int packs = hi > first ? (hi - first) / N : 0, tail = first + packs * N;
    if (lo >= hi) continue;  // (block-uniform)
    const int64_t t = tokens[token_at];
    const float m = stats[2 * row], ls2 = stats[2 * row + 1] * kLog2e;
    const float h = ENT ? g_ent[row] : 0.f, ent = ENT ? entropy[row] : 0.f;
    const float g = g_lp && t != ignore ? g_lp[row] : 0.f;
    const float g_own = lane < K ? g_top[row * K + lane] : 0.f;  // the alternatives' gradients, one to a lane
    float a = g + wave_sum(g_own);
    const bool any = g != 0.f || h != 0.f || __ballot(g_own != 0.f) != 0;
    if (!any || m == -INFINITY) {
      const float zero[N] = {};
#pragma unroll
      for (int i = 0; i < kBackPacks; ++i)
        if (i * THREADS + tid < packs) store_pack<T>(out + first + (i * THREADS + tid) * N, zero);
      if (lo + tid < first && lo + tid < hi) store_as(out + lo + tid, 0.f);
      if (tail + tid < hi) store_as(out + tail + tid, 0.f);
      continue;
    }
    if (g != 0.f && (t < 0 || t >= V)) a = quiet_nan();
    // d = x c - L and -p (a + h (d ln 2 + H)) / T = 2^d (c0 + c1 d)
    const float L = fmaf(m, c, ls2);
    const bool plain = __builtin_fabsf(L) < kPlainScale;
    const float rest_l = plain ? fmaf(m, c, -L) + ls2 : 0.f;  // L - its rounded value
    const float scale = -inv_t * __builtin_amdgcn_exp2f(-rest_l);
    const float c1 = ENT ? h * kLn2 * scale : 0.f;
    const float c0 = ENT ? scale * fmaf(h, fmaf(rest_l, -kLn2, ent), a) : scale * a;
    const auto power = [&](float v) { return plain ? fmaf(v, c, -L) : (v - m) * c - ls2; };
    const auto part = [&](float d) {
      const float p = __builtin_amdgcn_exp2f(d);
      return ENT ? p * fmaf(c1, fmaxf(d, -1000.f), c0) : p * c0;
    };
    const int64_t at = lane < K ? top_tok[row * K + lane] : -1;
    const bool mine = at >= lo && at < hi;
    const float x_own = mine ? load_as<T>(x + at) : 0.f, x_t = t >= lo && t < hi ? load_as<T>(x + t) : 0.f;
    u32x4 v[kBackPacks];
#pragma unroll
    for (int i = 0; i < kBackPacks; ++i)
      if (i * THREADS + tid < packs) v[i] = *reinterpret_cast<const u32x4_any*>(x + first + (i * THREADS + tid) * N);
#pragma unroll
    for (int i = 0; i < kBackPacks; ++i) {
      if (i * THREADS + tid < packs) {
        float o[N];
#pragma unroll
        for (int q = 0; q < N; ++q) o[q] = part(power(Pack<T>::get(v[i], q)));
        store_pack<T>(out + first + (i * THREADS + tid) * N, o);
      }
    }
    if (lo + tid < first && lo + tid < hi) store_as(out + lo + tid, part(power(load_as<T>(x + lo + tid))));
    if (tail + tid < hi) store_as(out + tail + tid, part(power(load_as<T>(x + tail + tid))));
    // The logits with a gradient of their own, each put over by the thread that has just written it.
    const auto owner_of = [&](int k) { return k < first ? k - lo : k < tail ? (k - first) / N % THREADS : k - tail; };
    const float value = fmaf(at == t ? g_own + g : g_own, inv_t, part(power(x_own)));
    const int k_own = (int)at, owner = owner_of(k_own);
    for (uint64_t left = __ballot(mine && owner >> 6 == tid >> 6); left; left &= left - 1) {
      const int i = __builtin_ctzll(left);
      const int k = __builtin_amdgcn_readlane(k_own, i);
      if (tid == __builtin_amdgcn_readlane(owner, i))
        store_as(out + k, __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(value), i)));
    }
    if (t >= lo && t < hi && __ballot(at == t) == 0 && tid == owner_of((int)t))
      store_as(out + t, fmaf(g, inv_t, part(power(x_t))));  // (else it is among the alternatives)
  }
}

constexpr int64_t kMaxBlocks = 1 << 20;  // rows of a launch that run at once
constexpr int64_t kMaxVocab = (int64_t)1 << 23;  // 1,024 segments of 8,192 fp32 logits

bool shape_ok(int64_t outer, int64_t inner, int64_t V, int64_t so, int64_t si) {
  return outer > 0 && inner > 0 && outer <= ((int64_t)1 << 40) / inner && V > 0 && V <= kMaxVocab && so >= 0 && si >= 0;
}

// The logits of a block: threads and packs of 16 bytes to each of them; segments of a row. One wave to a row that it
// holds (8,192 rows of 1,000 bf16: 7.2 us, 17.9 with four waves); 4 packs to a thread where they hold the row (4,096
// rows of 8,192: 14.1 us, 17.4 with 8 packs that half the threads fill) and 8 where they do not (8,192 rows of 16,384:
// 42 us in one segment, 64 in two of 4 packs). A row just above a block's logits is two segments that half fill it:
// 4,096 rows of 16,385 take 42 us and in three segments of 4 packs 40, of 20,000 42 and 43, of 32,768 54 and 56.
struct Tile {
  int threads, packs, segments;
  int64_t seg_len;
};

Tile tile_of(int64_t V, size_t size) {
  const int64_t n = (int64_t)(16 / size);
  if (V <= 64 * 4 * n) return {64, 4, 1, V};
  if (V <= 256 * 4 * n) return {256, 4, 1, V};
  const int64_t segments = cdiv(V, 256 * 8 * n), len = cdiv(cdiv(V, segments), n) * n;
  return {256, 8, (int)cdiv(V, len), len};
}

size_t part_bytes(int64_t rows, const Tile& tile, int64_t K) {
  return tile.segments == 1 ? 0 : (size_t)rows * tile.segments * (16 + 8 * K);
}

template <typename T>
int forward(const T* logits, const Rows& r, int64_t rows, int64_t V, float inv_t, const Outputs& out, void* workspace,
            const Tile& tile, hipStream_t s) {
  const dim3 grid((unsigned)(rows < kMaxBlocks ? rows : kMaxBlocks), (unsigned)tile.segments);
  f32x4* part = static_cast<f32x4*>(workspace);
  uint64_t* keys = reinterpret_cast<uint64_t*>(part + (tile.segments == 1 ? 0 : rows * tile.segments));
#define FL_LP2(N, P, ENT, TOP)                                                                                     \
  fl_token_logprobs_kernel<T, N, P, ENT, TOP><<<grid, N, 0, s>>>(logits, r, rows, (int)V, (int)tile.seg_len, inv_t, \
                                                                 out, part, keys)
#define FL_LP(N, P)                                                                                                \
  if (tile.threads == N && tile.packs == P) {                                                                      \
    if (out.entropy && out.K) FL_LP2(N, P, true, true);                                                            \
    else if (out.entropy) FL_LP2(N, P, true, false);                                                               \
    else if (out.K) FL_LP2(N, P, false, true);                                                                     \
    else FL_LP2(N, P, false, false);                                                                               \
  }
  FL_LP(64, 4)
  FL_LP(256, 4)
  FL_LP(256, 8)
#undef FL_LP
#undef FL_LP2
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || tile.segments == 1) return hip_status(e);
  if (tile.segments <= 64)
    fl_token_logprobs_join_kernel<T, 256, true><<<grid.x, 256, 0, s>>>(logits, r, rows, (int)V, tile.segments, inv_t,
                                                                       out, part, keys);
  else
    fl_token_logprobs_join_kernel<T, 1024, false><<<grid.x, 1024, 0, s>>>(logits, r, rows, (int)V, tile.segments,
                                                                          inv_t, out, part, keys);
  return hip_status(hipGetLastError());
}

}  // namespace

extern "C" {

size_t fl_token_logprobs_workspace_bytes(int64_t rows, int64_t V, int dtype, int64_t top_k) {
  if (rows <= 0 || rows > (int64_t)1 << 40 || V <= 0 || V > kMaxVocab || top_k < 0 || top_k > kMaxTop) return 0;
  if (!dtype_ok(dtype)) return 0;
  return part_bytes(rows, tile_of(V, esize(dtype)), top_k);
}

int fl_token_logprobs(const void* logits, int dtype, int64_t outer, int64_t inner, int64_t V, int64_t stride_outer,
                      int64_t stride_inner, const int64_t* tokens, int64_t token_outer, int64_t token_inner,
                      int64_t ignore_index, float temperature, int64_t top_k, float* logprobs, float* entropy,
                      float* top_logprobs, int64_t* top_tokens, float* stats, void* workspace, size_t workspace_bytes,
                      void* stream) {
  if (!dtype_ok(dtype)) return FL_ERR_DTYPE;
  if (!shape_ok(outer, inner, V, stride_outer, stride_inner) ||
      !(temperature >= kMinTemperature && temperature <= kMaxTemperature) ||
      top_k < 0 || top_k > kMaxTop || top_k > V)
    return FL_ERR_INVALID_ARGUMENT;
  if (!logits || !aligned(logits, esize(dtype)) || !tokens || !aligned(tokens, 8) || !logprobs ||
      !aligned(logprobs, 4) || !aligned(entropy, 4) || !aligned(stats, 4) ||
      (top_k && (!top_logprobs || !top_tokens || !aligned(top_logprobs, 4) || !aligned(top_tokens, 8))))
    return FL_ERR_INVALID_ARGUMENT;
  const int64_t rows = outer * inner;
  const Tile tile = tile_of(V, esize(dtype));
  const size_t need = part_bytes(rows, tile, top_k);
  if (need && (!workspace || workspace_bytes < need)) return FL_ERR_WORKSPACE;
  if (need && !aligned(workspace, 16)) return FL_ERR_INVALID_ARGUMENT;
  const Rows r = {inner, stride_outer, stride_inner, token_outer, token_inner};
  const Outputs out = {tokens, ignore_index, (int)top_k, logprobs, entropy, top_logprobs, top_tokens, stats};
  hipStream_t s = static_cast<hipStream_t>(stream);
  const float inv_t = 1.0f / temperature;
  return dtype == FL_DTYPE_BF16
             ? forward(static_cast<const bf16_bits*>(logits), r, rows, V, inv_t, out, workspace, tile, s)
             : forward(static_cast<const float*>(logits), r, rows, V, inv_t, out, workspace, tile, s);
}

int fl_token_logprobs_backward(const void* logits, int dtype, int64_t outer, int64_t inner, int64_t V,
                               int64_t stride_outer, int64_t stride_inner, const int64_t* tokens, int64_t token_outer,
                               int64_t token_inner, int64_t ignore_index, float temperature, int64_t top_k,
                               const float* stats, const float* entropy, const int64_t* top_tokens,
                               const float* g_logprobs, const float* g_entropy, const float* g_top, void* g_logits,
                               void* stream) {
  if (!dtype_ok(dtype)) return FL_ERR_DTYPE;
  if (!shape_ok(outer, inner, V, stride_outer, stride_inner) ||
      !(temperature >= kMinTemperature && temperature <= kMaxTemperature) ||
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
  // one wave to a row that it holds, four otherwise (8,192 rows of 1,000 bf16: 9.6 us, with four waves 15.8)
  const int64_t pack = (int64_t)(kBackPacks * 16 / esize(dtype));
  const int threads = V <= 64 * pack ? 64 : 256;
  const dim3 grid((unsigned)blocks, (unsigned)cdiv(V, threads * pack));
#define FL_LB2(T, N, ENT)                                                                                          \
  fl_token_logprobs_backward_kernel<T, N, ENT><<<grid, N, 0, s>>>(                                                 \
      static_cast<const T*>(logits), r, rows, (int)V, tokens, ignore_index, 1.0f / temperature,                    \
      g_top ? (int)top_k : 0, stats, entropy, top_tokens, g_logprobs, g_entropy, g_top, static_cast<T*>(g_logits))
#define FL_LB(T)                                                                                                   \
  if (threads == 64 && g_entropy) FL_LB2(T, 64, true);                                                             \
  else if (threads == 64) FL_LB2(T, 64, false);                                                                    \
  else if (g_entropy) FL_LB2(T, 256, true);                                                                        \
  else FL_LB2(T, 256, false);
  if (dtype == FL_DTYPE_BF16) {
    FL_LB(bf16_bits)
  } else {
    FL_LB(float)
  }
#undef FL_LB2
#undef FL_LB
  return hip_status(hipGetLastError());
}

}  // extern "C"
