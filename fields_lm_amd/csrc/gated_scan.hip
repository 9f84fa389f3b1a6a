// gated_scan.hip — the gated linear recurrence over T steps and its gradients:
//   h_t = a_t h_{t-1} + u_t,  h_{-1} = state_in or 0,          a gate to every channel or one to a token;
//   g_t = dh_t + a_{t+1} g_{t+1}  (the last step's carry is the final state's gradient),
//   du_t = g_t,  da_t = g_t h_{t-1} (summed over the channels where they share a gate),  dstate_in = a_0 g_0.
//
// A run of steps is a map h -> P h + S (P the product of its gates, S its end from 0), and maps compose; the reverse
// recurrence's maps have the same P. A block takes a tile of 256 steps and 64 channels and holds it in registers, 16 lanes
// with four channels each to a segment of consecutive steps. It composes its segments' maps through the LDS, gets the
// tile's start from the tiles before it, and runs its steps from there: inputs are read once. The backward pass forms the
// states again from each tile's start, which the forward pass keeps (4 bytes to 256 steps), in place of reading them:
// those are rounded to the drive's type, and cost as much to read as the drive.
//
// Tiles of a chain (a sequence's 64 channels) find their start by looking back: each publishes its map, then its end, as
// words of a value and a mark that it is there, and takes the maps of those before it up to the first that has
// published its end. Tiles are taken in the order in which blocks start, from a counter: a tile waits only for tiles that
// are running or done, so that every wait ends. The words are cleared by a launch before.
//
// Bound by memory, in rounds of blocks that read, wait and write in turn: B=8, T=2,048, C=1,024 in fp32 47 us forward
// (4.3 TB/s) and 68 us back (5.0 TB/s); B=1, T=65,536, fp32 gates and bf16 drives 106 us (5.1 TB/s) and 185 us (5.1 TB/s),
// where three launches over the same tiles (maps, composition, steps) took 2.8 ms. Of the forward's blocks with a gate a channel two fit a CU (190 registers a lane), by a limit: with
// three more tiles look back at once and further (42.5 us for the first in place of 39.5 without gradients kept). With a
// gate a token four do (126), and of the backward's blocks, twice as many threads, one does (158 and 128).
#include "fl_common.h"

#include <type_traits>

namespace {

using namespace fl;

constexpr int kTile = 256;     // steps
constexpr int kChannels = 64;  // of a chain
constexpr int kWords = 3 * kChannels;  // of a tile: P and S of its map, its end
constexpr int kShort = 8;      // steps up to which no tile is formed (64 sequences of 1,024 channels, one step: 3.2 us, a
                               // tile each 8.1)
constexpr int kHeld = 16;      // tiles whose maps a tile holds; it waits for an end where it would need more
constexpr uint32_t kMaxPolls = 1u << 20;  // of a wait that never ends; its tile's results are NaN
constexpr int64_t kMaxB = 1 << 24, kMaxC = 1 << 24, kMaxT = (int64_t)1 << 30;

struct Scan {
  const void* gate;
  const void* drive;
  int64_t gate_b, gate_t, drive_b, drive_t;  // strides in elements
  int64_t T, C;
  int tiles, groups;   // of a chain, of 64 channels
  unsigned chains;
  uint32_t* ticket;    // null where chains have one tile
  uint64_t* words;     // [tiles, chains, kWords]
};

// four values of a row as they lie, `left` of them there
template <typename T>
struct Four;
template <>
struct Four<float> {
  float v[4];
  __device__ __forceinline__ void load(const float* p, int64_t left) {
    if (left >= 4) {
      const u32x4 r = *reinterpret_cast<const u32x4_any*>(p);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(r[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = i < left ? p[i] : 0.f;
    }
  }
  __device__ __forceinline__ void fill(float x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = x;
  }
  __device__ __forceinline__ float operator[](int i) const { return v[i]; }
};
template <>
struct Four<bf16_bits> {
  uint32_t w[2];
  __device__ __forceinline__ void load(const bf16_bits* p, int64_t left) {
    if (left >= 4) {
      const u32x2 r = *reinterpret_cast<const u32x2_any*>(p);
      w[0] = r[0];
      w[1] = r[1];
    } else {
      w[0] = w[1] = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i < left) w[i >> 1] |= (uint32_t)p[i] << (16 * (i & 1));
    }
  }
  __device__ __forceinline__ void fill(float x) { w[0] = w[1] = bf16_bits_of(x) * 0x10001u; }
  __device__ __forceinline__ float operator[](int i) const { return i & 1 ? bf16_hi(w[i >> 1]) : bf16_lo(w[i >> 1]); }
};
// Streaming stores: 11% less time for B=8, T=2,048, C=1,024 in fp32 with gradients, 2% for B=1, T=65,536; what reads the result
// next is as fast behind either (2 to 270 MB).
__device__ __forceinline__ void store4(float* p, int64_t left, const float* v) {
  if (left >= 4) {
    const u32x4 r = {__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
    __builtin_nontemporal_store(r, reinterpret_cast<u32x4_any*>(p));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < left) p[i] = v[i];
  }
}
__device__ __forceinline__ void store4(bf16_bits* p, int64_t left, const float* v) {
  if (left >= 4) {
    const u32x2 r = {bf16_pair(v[0], v[1]), bf16_pair(v[2], v[3])};
    __builtin_nontemporal_store(r, reinterpret_cast<u32x2_any*>(p));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < left) store_as(p + i, v[i]);
  }
}

// lane J of each 16 in all of them (every lane has to be there)
template <int J>
__device__ __forceinline__ float of_lane(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x150 + J, 0xf, 0xf, true));
}
// the sum over each 16 lanes, in all of them
__device__ __forceinline__ float row_sum(float v) {
  v = dpp_add<0xb1>(v);
  v = dpp_add<0x4e>(v);
  v = dpp_add<0x141>(v);
  return dpp_add<0x140>(v);
}

// The gates of a segment's STEPS steps: a value to every channel, or (TOKEN) one to a step, held by the lane of its number.
template <typename GT, bool TOKEN, int STEPS>
struct Gates;
template <typename GT, int STEPS>
struct Gates<GT, false, STEPS> {
  Four<GT> v[STEPS];
  __device__ __forceinline__ void load(const GT* p, int64_t step, int n, int, int64_t left) {
#pragma unroll
    for (int j = 0; j < STEPS; ++j) {
      v[j].fill(1.f);
      if (j < n && left > 0) v[j].load(p + j * step, left);
    }
  }
  template <int J>
  __device__ __forceinline__ float at(int i) const { return v[J][i]; }
};
template <typename GT, int STEPS>
struct Gates<GT, true, STEPS> {
  float v;
  __device__ __forceinline__ void load(const GT* p, int64_t step, int n, int lane, int64_t) {
    v = lane < n ? load_as<GT>(p + lane * step) : 1.f;
  }
  template <int J>
  __device__ __forceinline__ float at(int) const { return of_lane<J>(v); }
};

// A run's product of gates is held in fp64: in fp32 that of ordinary ones leaves the range (0.5^256), and a large state, or
// gates above 1 that follow, would bring what is lost of it back. One too small for that too is kept off 0, which is a
// closed gate's alone: an infinite state before such a run is infinite behind it, as it is step by step, and a finite
// one passes nothing (2^-1022 of it). One too large is kept finite, so that a state of 0 passes 0 and any other infinity.
// The last bit stays clear, for `publish`.
constexpr double kLeast = 0x1p-1022, kMost = 0x1.ffffffffffffep1023;
__device__ __forceinline__ double kept(double product, bool closed) {
  const double size = fmin(fmax(fabs(product), kLeast), kMost);
  return closed ? 0.0 : __longlong_as_double(__double_as_longlong(copysign(size, product)) & ~1ll);
}

template <int N, int I = 0, typename F>
__device__ __forceinline__ void each(F f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>());
    each<N, I + 1>(f);
  }
}
template <int N, typename F>
__device__ __forceinline__ void each_back(F f) {
  each<N>([&](auto i) { f(std::integral_constant<int, N - 1 - decltype(i)::value>()); });
}

// a word: the last bit says that it is there, the others are a product's, or a float's in the upper half
__device__ __forceinline__ void publish(uint64_t* to, uint64_t bits) {
  __hip_atomic_store(to, bits | 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void publish(uint64_t* to, float v) { publish(to, (uint64_t)__float_as_uint(v) << 32); }
__device__ __forceinline__ void publish(uint64_t* to, double p) { publish(to, (uint64_t)__double_as_longlong(p)); }
__device__ __forceinline__ uint64_t published(const uint64_t* from) {
  return __hip_atomic_load(from, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ bool there(uint64_t w) { return __all(w & 1u); }
__device__ __forceinline__ float value_of(uint64_t w) { return __uint_as_float((uint32_t)(w >> 32)); }
__device__ __forceinline__ double product_of(uint64_t w) { return __longlong_as_double((long long)(w & ~(uint64_t)1)); }

// a state behind a run
__device__ __forceinline__ double through(double p, double h, double s) { return fma(p, h, s); }

// What enters a tile behind its chain's first: the end of the nearest tile before it that has published one, through
// the maps of those between, which are held in `hold_p` and `hold_s` (kHeld rows of kChannels, the lane's column). Each
// map is applied as its own tile applies it, so that the bits are the same wherever an end was found (one product of the
// maps took 2 us less of 286, with bits that varied). `words`: the
// tile's own, lane's channel; `back`: words from a tile to the one before it.
__device__ __forceinline__ float look_back(const uint64_t* words, int64_t back, double* hold_p, float* hold_s) {
  uint32_t polls = 0;
  for (int i = 0;;) {
    words -= back;  // (the first tile of a chain has an end, and is the last to be looked at)
    uint64_t p, s, end;
    for (;;) {
      p = published(words);
      s = published(words + kChannels);
      end = published(words + 2 * kChannels);
      if (there(end) || (i < kHeld && there(p) && there(s))) break;
      if (++polls >= kMaxPolls) return __uint_as_float(0x7fc00000u);
      __builtin_amdgcn_s_sleep(1);
    }
    if (there(end)) {
      float h = value_of(end);
      for (; i > 0; --i) h = (float)through(hold_p[(i - 1) * kChannels], h, hold_s[(i - 1) * kChannels]);
      return h;
    }
    hold_p[i * kChannels] = product_of(p);
    hold_s[i * kChannels] = value_of(s);
    ++i;
  }
}

// What enters a tile's segments: `first` through the products of those before each (BACK: behind each), whose ends are in
// `ends`. The products are the bare ones, which may have left fp64: a state of 0 passes none, and for an infinite one, in its
// own lane, they are formed again.
template <int SEGS, bool BACK>
__device__ __forceinline__ void enter(const double (*each_p)[kChannels], const double (*run_p)[kChannels],
                                      float (*ends)[kChannels], int ch, float first) {
  if (fabsf(first) == __builtin_inff()) {
    double run = 1.0;
    for (int i = 0; i < SEGS; ++i) {
      const int seg = BACK ? SEGS - 1 - i : i;
      ends[seg][ch] = (float)through(run, first, ends[seg][ch]);
      run = kept(run * each_p[seg][ch], run == 0.0 || each_p[seg][ch] == 0.0);
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < SEGS; ++i) {
    const float end = ends[i][ch], now = (float)through(run_p[i][ch], first, end);
    ends[i][ch] = first == 0.f ? end : now;
  }
}

// Where a block's tile lies
struct Place {
  int place, tile;  // in the order of the scan, in time
  unsigned chain;
  int64_t b, c0;
  bool there;
};
template <bool BACK>
__device__ __forceinline__ Place place_of(const Scan& s, uint32_t* s_ticket) {
  unsigned t = blockIdx.y * gridDim.x + blockIdx.x;
  if (s.ticket) {
    if (threadIdx.x == 0)
      *s_ticket = __hip_atomic_fetch_add(s.ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    t = (unsigned)uniform((int)*s_ticket);
  }
  Place r;
  r.there = t < (unsigned)s.tiles * s.chains;
  r.place = (int)(t / s.chains);
  r.chain = t - (unsigned)r.place * s.chains;
  r.tile = BACK ? s.tiles - 1 - r.place : r.place;
  r.b = r.chain / (unsigned)s.groups;
  r.c0 = (int64_t)(r.chain - (unsigned)r.b * (unsigned)s.groups) * kChannels;
  return r;
}

constexpr int kForwardSteps = 16, kBackSteps = 8;  // of a segment
constexpr int kForwardThreads = kTile / kForwardSteps * 16, kBackThreads = kTile / kBackSteps * 16;

template <typename GT, typename DT, bool TOKEN>
__global__ __launch_bounds__(kForwardThreads) __attribute__((amdgpu_waves_per_eu(2, TOKEN ? 4 : 2)))
void fl_gated_scan_kernel(const Scan s, const float* __restrict__ state_in,
                                                                        float* __restrict__ state_out,
                                                                        float* __restrict__ starts,
                                                                        DT* __restrict__ out) {
  constexpr int STEPS = kForwardSteps, SEGS = kTile / STEPS;
  __shared__ double s_p[SEGS][kChannels], s_before[SEGS][kChannels], s_hold_p[kHeld][kChannels];
  __shared__ float s_s[SEGS][kChannels], s_hold_s[kHeld][kChannels];
  __shared__ uint32_t s_ticket;
  const Place at = place_of<false>(s, &s_ticket);
  if (!at.there) return;  // (the whole block)
  const int seg = threadIdx.x >> 4, lane = threadIdx.x & 15;
  const int64_t c = at.c0 + lane * 4, left = s.C - c, t0 = (int64_t)at.tile * kTile + seg * STEPS;
  const int n = (int)(s.T - t0 < STEPS ? (s.T > t0 ? s.T - t0 : 0) : STEPS);
  Gates<GT, TOKEN, STEPS> a;
  Four<DT> u[STEPS];
  a.load(static_cast<const GT*>(s.gate) + at.b * s.gate_b + t0 * s.gate_t + (TOKEN ? 0 : c), s.gate_t, n, lane, left);
  const DT* from = static_cast<const DT*>(s.drive) + at.b * s.drive_b + t0 * s.drive_t + c;
#pragma unroll
  for (int j = 0; j < STEPS; ++j) {
    u[j].fill(0.f);
    if (j < n && left > 0) u[j].load(from + j * s.drive_t, left);
  }
  double p[4] = {1.0, 1.0, 1.0, 1.0};
  f32x4 least = {1.f, 1.f, 1.f, 1.f}, h = {0.f, 0.f, 0.f, 0.f};
  each<STEPS>([&](auto j) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float g = a.template at<decltype(j)::value>(i);
      h[i] = fmaf(g, h[i], u[decltype(j)::value][i]);
      p[i] *= g;
      least[i] = fminf(least[i], fabsf(g));
    }
  });
#pragma unroll
  for (int i = 0; i < 4; ++i) s_p[seg][lane * 4 + i] = kept(p[i], least[i] == 0.f);
  *reinterpret_cast<f32x4*>(&s_s[seg][lane * 4]) = h;
  __syncthreads();
  if (threadIdx.x < kChannels) {
    const int ch = threadIdx.x;
    const int64_t k = at.c0 + ch;
    double run = 1.0, smallest = 1.0, end = 0.0;
#pragma unroll
    for (int i = 0; i < SEGS; ++i) {
      const double pi = s_p[i][ch];
      const float si = s_s[i][ch];
      s_before[i][ch] = run;
      s_s[i][ch] = (float)end;
      end = through(pi, end, si);
      run *= pi;
      smallest = fmin(smallest, fabs(pi));
    }
    const double pt = kept(run, smallest == 0.0);
    const float st = (float)end;
    uint64_t* words = s.words + ((int64_t)at.place * s.chains + at.chain) * kWords + ch;
    float first;
    const bool more = at.place + 1 < s.tiles;
    if (at.place == 0) {
      first = state_in && k < s.C ? state_in[at.b * s.C + k] : 0.f;
    } else {
      if (more) {
        publish(words, pt);
        publish(words + kChannels, st);
      }
      first = look_back(words, (int64_t)s.chains * kWords, &s_hold_p[0][ch], &s_hold_s[0][ch]);
    }
    const float last = (float)through(pt, first, st);
    if (more) publish(words + 2 * kChannels, last);
    enter<SEGS, false>(s_p, s_before, s_s, ch, first);
    if (k < s.C) {
      if (starts) starts[(at.b * s.tiles + at.tile) * s.C + k] = first;
      if (state_out && !more) state_out[at.b * s.C + k] = last;
    }
  }
  __syncthreads();
  h = *reinterpret_cast<const f32x4*>(&s_s[seg][lane * 4]);
  DT* to = out + (at.b * s.T + t0) * s.C + c;
  each<STEPS>([&](auto j) {
    float v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      h[i] = fmaf(a.template at<decltype(j)::value>(i), h[i], u[decltype(j)::value][i]);
      v[i] = h[i];
    }
    if (decltype(j)::value < n && left > 0) store4(to + decltype(j)::value * s.C, left, v);
  });
}

// A few steps: 16 lanes to a chain, step by step.
template <typename GT, typename DT, bool TOKEN>
__global__ __launch_bounds__(256) void fl_gated_short_kernel(const Scan s, const float* __restrict__ state_in,
                                                             float* __restrict__ state_out, float* __restrict__ starts,
                                                             DT* __restrict__ out) {
  constexpr int STEPS = kShort;
  const unsigned chain = (blockIdx.y * gridDim.x + blockIdx.x) * 16 + (threadIdx.x >> 4);
  const int lane = threadIdx.x & 15;
  const int64_t b = chain / (unsigned)s.groups, c0 = (int64_t)(chain - (unsigned)b * (unsigned)s.groups) * kChannels;
  const int64_t c = c0 + lane * 4, left = s.C - c;
  const int n = chain < s.chains ? (int)s.T : 0;
  Gates<GT, TOKEN, STEPS> a;
  Four<DT> u[STEPS];
  Four<float> h;
  a.load(static_cast<const GT*>(s.gate) + b * s.gate_b + (TOKEN ? 0 : c), s.gate_t, n, lane, left);
  const DT* from = static_cast<const DT*>(s.drive) + b * s.drive_b + c;
#pragma unroll
  for (int j = 0; j < STEPS; ++j) {
    u[j].fill(0.f);
    if (j < n && left > 0) u[j].load(from + j * s.drive_t, left);
  }
  h.fill(0.f);
  const bool ok = n > 0 && left > 0;
  if (ok && state_in) h.load(state_in + b * s.C + c, left);
  if (ok && starts) store4(starts + b * s.C + c, left, h.v);
  DT* to = out + b * s.T * s.C + c;
  each<STEPS>([&](auto j) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      h.v[i] = fmaf(a.template at<decltype(j)::value>(i), h.v[i], u[decltype(j)::value][i]);
    if (decltype(j)::value < n && left > 0) store4(to + decltype(j)::value * s.C, left, h.v);
  });
  if (ok && state_out) store4(state_out + b * s.C + c, left, h.v);
}

// Wave 0 composes the tile's maps forward from the state it starts from, wave 1 backward from the carry into its end.
template <typename GT, typename DT, bool TOKEN>
__global__ __launch_bounds__(kBackThreads) void fl_gated_back_kernel(
    const Scan s, const float* __restrict__ starts, const DT* __restrict__ g_out, const float* __restrict__ g_state,
    GT* __restrict__ g_gate, float* __restrict__ part, DT* __restrict__ g_drive, float* __restrict__ g_state_in) {
  constexpr int STEPS = kBackSteps, SEGS = kTile / STEPS;
  __shared__ double s_p[SEGS][kChannels], s_after[SEGS][kChannels], s_hold_p[kHeld][kChannels];
  __shared__ float s_h[SEGS][kChannels], s_k[SEGS][kChannels], s_hold_k[kHeld][kChannels];
  __shared__ uint32_t s_ticket;
  const Place at = place_of<true>(s, &s_ticket);
  if (!at.there) return;  // (the whole block)
  const int seg = threadIdx.x >> 4, lane = threadIdx.x & 15;
  const int64_t c = at.c0 + lane * 4, left = s.C - c, t0 = (int64_t)at.tile * kTile + seg * STEPS;
  const int n = (int)(s.T - t0 < STEPS ? (s.T > t0 ? s.T - t0 : 0) : STEPS);
  Gates<GT, TOKEN, STEPS> a;
  Four<DT> u[STEPS], d[STEPS];
  a.load(static_cast<const GT*>(s.gate) + at.b * s.gate_b + t0 * s.gate_t + (TOKEN ? 0 : c), s.gate_t, n, lane, left);
  const DT* from = static_cast<const DT*>(s.drive) + at.b * s.drive_b + t0 * s.drive_t + c;
  const DT* up = g_out + (at.b * s.T + t0) * s.C + c;
#pragma unroll
  for (int j = 0; j < STEPS; ++j) {
    d[j].fill(0.f);
    if (g_out && j < n && left > 0) d[j].load(up + j * s.C, left);
  }
#pragma unroll
  for (int j = 0; j < STEPS; ++j) {
    u[j].fill(0.f);
    if (j < n && left > 0) u[j].load(from + j * s.drive_t, left);
  }
  double p[4] = {1.0, 1.0, 1.0, 1.0};
  f32x4 least = {1.f, 1.f, 1.f, 1.f}, h = {0.f, 0.f, 0.f, 0.f}, k = h;
  each<STEPS>([&](auto j) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float g = a.template at<decltype(j)::value>(i);
      h[i] = fmaf(g, h[i], u[decltype(j)::value][i]);
      p[i] *= g;
      least[i] = fminf(least[i], fabsf(g));
    }
  });
#pragma unroll
  for (int i = 0; i < 4; ++i) s_p[seg][lane * 4 + i] = kept(p[i], least[i] == 0.f);
  each_back<STEPS>([&](auto j) {
#pragma unroll
    for (int i = 0; i < 4; ++i) k[i] = a.template at<decltype(j)::value>(i) * (k[i] + d[decltype(j)::value][i]);
  });
  *reinterpret_cast<f32x4*>(&s_h[seg][lane * 4]) = h;
  *reinterpret_cast<f32x4*>(&s_k[seg][lane * 4]) = k;
  __syncthreads();
  const int ch = threadIdx.x & 63;
  const int64_t cc = at.c0 + ch;
  if (threadIdx.x < 64) {
    double now = cc < s.C ? starts[(at.b * s.tiles + at.tile) * s.C + cc] : 0.f;
#pragma unroll
    for (int i = 0; i < SEGS; ++i) {
      const float hi = s_h[i][ch];
      s_h[i][ch] = (float)now;
      now = through(s_p[i][ch], now, hi);
    }
  } else if (threadIdx.x < 128) {
    double run = 1.0, smallest = 1.0, end = 0.0;
#pragma unroll
    for (int i = SEGS - 1; i >= 0; --i) {
      const double pi = s_p[i][ch];
      const float ki = s_k[i][ch];
      s_after[i][ch] = run;
      s_k[i][ch] = (float)end;
      end = through(pi, end, ki);
      run *= pi;
      smallest = fmin(smallest, fabs(pi));
    }
    const double pt = kept(run, smallest == 0.0);
    const float kt = (float)end;
    uint64_t* words = s.words + ((int64_t)at.place * s.chains + at.chain) * kWords + ch;
    float first;
    const bool more = at.place + 1 < s.tiles;
    if (at.place == 0) {
      first = g_state && cc < s.C ? g_state[at.b * s.C + cc] : 0.f;
    } else {
      if (more) {
        publish(words, pt);
        publish(words + kChannels, kt);
      }
      first = look_back(words, (int64_t)s.chains * kWords, &s_hold_p[0][ch], &s_hold_k[0][ch]);
    }
    const float last = (float)through(pt, first, kt);
    if (more) publish(words + 2 * kChannels, last);
    enter<SEGS, true>(s_p, s_after, s_k, ch, first);
    if (g_state_in && !more && cc < s.C) g_state_in[at.b * s.C + cc] = last;
  }
  __syncthreads();
  h = *reinterpret_cast<const f32x4*>(&s_h[seg][lane * 4]);
  k = *reinterpret_cast<const f32x4*>(&s_k[seg][lane * 4]);
  f32x4 before[STEPS];
  each<STEPS>([&](auto j) {
    before[decltype(j)::value] = h;
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = fmaf(a.template at<decltype(j)::value>(i), h[i], u[decltype(j)::value][i]);
  });
  const int64_t row = at.b * s.T + t0;
  each_back<STEPS>([&](auto jj) {
    constexpr int j = decltype(jj)::value;
    float g[4], da[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      g[i] = d[j][i] + k[i];
      da[i] = g[i] * before[j][i];
      k[i] = a.template at<j>(i) * g[i];
    }
    if (j < n && left > 0) store4(g_drive + (row + j) * s.C + c, left, g);
    if constexpr (TOKEN) {
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) sum += i < left ? da[i] : 0.f;
      sum = row_sum(sum);
      if (g_gate && j < n && lane == 0) {
        if (s.groups == 1)
          store_as(g_gate + row + j, sum);
        else
          part[(at.c0 / kChannels) * ((int64_t)(s.chains / (unsigned)s.groups) * s.T) + row + j] = sum;
      }
    } else {
      if (g_gate && j < n && left > 0) store4(g_gate + (row + j) * s.C + c, left, da);
    }
  });
}

__global__ __launch_bounds__(256) void fl_gated_clear_kernel(u32x4* __restrict__ p, int64_t n) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) p[i] = u32x4{0, 0, 0, 0};
}

// the gradient of a token's gate: the sums of its groups of channels, in their order
template <typename GT>
__global__ __launch_bounds__(256) void fl_gated_token_kernel(const float* __restrict__ part, int64_t n, int groups,
                                                             GT* __restrict__ g_gate) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  float sum = 0.f;
  for (int k = 0; k < groups; ++k) sum += part[k * n + i];
  store_as(g_gate + i, sum);
}

struct Call {
  Scan s;
  int64_t B;
  hipStream_t stream;
};

// rows of 2^22 blocks: a row's threads have to be fewer than 2^32
dim3 grid_of(int64_t blocks) {
  const int64_t row = (int64_t)1 << 22;
  return blocks <= row ? dim3((unsigned)blocks) : dim3((unsigned)row, (unsigned)cdiv(blocks, row));
}

// bytes of the ticket's line and the words; 0 where chains have one tile
size_t word_bytes(int64_t B, int64_t T, int64_t C) {
  const int64_t tiles = cdiv(T, kTile);
  return tiles > 1 ? 128 + (size_t)(tiles * B * cdiv(C, kChannels)) * kWords * 8 : 0;
}

void clear(const Call& c, size_t bytes) {
  if (!c.s.ticket) return;
  const int64_t n = (int64_t)(bytes / 16);
  const unsigned blocks = (unsigned)(cdiv(n, 256) < 2048 ? cdiv(n, 256) : 2048);
  fl_gated_clear_kernel<<<blocks, 256, 0, c.stream>>>(reinterpret_cast<u32x4*>(c.s.ticket), n);
}

template <typename GT, typename DT, bool TOKEN>
int forward(const Call& c, size_t bytes, const float* state_in, float* state_out, float* starts, void* out) {
  if (c.s.T <= kShort) {
    fl_gated_short_kernel<GT, DT, TOKEN><<<grid_of(cdiv((int64_t)c.s.chains, (int64_t)16)), 256, 0, c.stream>>>(
        c.s, state_in, state_out, starts, static_cast<DT*>(out));
    return hip_status(hipGetLastError());
  }
  clear(c, bytes);
  fl_gated_scan_kernel<GT, DT, TOKEN><<<grid_of((int64_t)c.s.tiles * c.s.chains), kForwardThreads, 0, c.stream>>>(c.s, state_in, state_out, starts,
                                                                                     static_cast<DT*>(out));
  return hip_status(hipGetLastError());
}

template <typename GT, typename DT, bool TOKEN>
int backward(const Call& c, size_t bytes, const float* starts, const void* g_out, const float* g_state, void* g_gate,
             void* g_drive, float* g_state_in, float* part) {
  clear(c, bytes);
  fl_gated_back_kernel<GT, DT, TOKEN><<<grid_of((int64_t)c.s.tiles * c.s.chains), kBackThreads, 0, c.stream>>>(
      c.s, starts, static_cast<const DT*>(g_out), g_state, static_cast<GT*>(g_gate), part, static_cast<DT*>(g_drive),
      g_state_in);
  if (TOKEN && g_gate && c.s.groups > 1) {
    const int64_t n = c.B * c.s.T;
    fl_gated_token_kernel<GT><<<(unsigned)cdiv(n, 256), 256, 0, c.stream>>>(part, n, c.s.groups,
                                                                            static_cast<GT*>(g_gate));
  }
  return hip_status(hipGetLastError());
}

bool sizes_ok(int64_t B, int64_t T, int64_t C) {
  return B > 0 && T > 0 && C > 0 && B <= kMaxB && C <= kMaxC && T <= kMaxT &&
         cdiv(T, kTile) * B <= (((int64_t)1 << 31) - 1) / cdiv(C, kChannels) &&  // blocks of a launch
         T * B <= ((int64_t)1 << 40) / C;
}

bool tensor_ok(const void* p, int dtype, int64_t stride_b, int64_t stride_t) {
  return p && aligned(p, esize(dtype)) && stride_b >= 0 && stride_t >= 0;
}

// a call without a workspace's need takes any
bool workspace_ok(const void* workspace, size_t have, size_t need) { return need == 0 || (workspace && have >= need); }

Call call_of(const void* gate, int64_t gate_b, int64_t gate_t, const void* drive, int64_t drive_b, int64_t drive_t,
             int64_t B, int64_t T, int64_t C, void* workspace, void* stream) {
  Call c = {};
  const bool one = cdiv(T, kTile) == 1;
  c.s = Scan{gate, drive, gate_b, gate_t, drive_b, drive_t, T, C, (int)cdiv(T, kTile), (int)cdiv(C, kChannels),
             (unsigned)(B * cdiv(C, kChannels)), one ? nullptr : static_cast<uint32_t*>(workspace),
             one ? nullptr : reinterpret_cast<uint64_t*>(static_cast<char*>(workspace) + 128)};
  c.B = B;
  c.stream = static_cast<hipStream_t>(stream);
  return c;
}

}  // namespace

extern "C" {

int64_t fl_gated_scan_tile(void) { return kTile; }

size_t fl_gated_scan_workspace_bytes(int64_t B, int64_t T, int64_t C, int backward) {
  if (!sizes_ok(B, T, C)) return 0;
  const int64_t groups = cdiv(C, kChannels);
  return word_bytes(B, T, C) + (backward && groups > 1 ? (size_t)(groups * B * T) * 4 : 0);
}

#define FL_GATED(CALL, ...)                                                                        \
  const bool a16 = gate_dtype == FL_DTYPE_BF16, u16 = drive_dtype == FL_DTYPE_BF16;                \
  if (per_token) {                                                                                 \
    if (a16) return u16 ? CALL<bf16_bits, bf16_bits, true>(__VA_ARGS__) : CALL<bf16_bits, float, true>(__VA_ARGS__); \
    return u16 ? CALL<float, bf16_bits, true>(__VA_ARGS__) : CALL<float, float, true>(__VA_ARGS__); \
  }                                                                                                \
  if (a16) return u16 ? CALL<bf16_bits, bf16_bits, false>(__VA_ARGS__) : CALL<bf16_bits, float, false>(__VA_ARGS__); \
  return u16 ? CALL<float, bf16_bits, false>(__VA_ARGS__) : CALL<float, float, false>(__VA_ARGS__);

int fl_gated_scan(const void* gate, int gate_dtype, int per_token, int64_t gate_stride_b, int64_t gate_stride_t,
                  const void* drive, int drive_dtype, int64_t drive_stride_b, int64_t drive_stride_t, int64_t B,
                  int64_t T, int64_t C, const float* state_in, float* state_out, float* starts, void* out,
                  void* workspace, size_t workspace_bytes, void* stream) {
  if (!dtype_ok(gate_dtype) || !dtype_ok(drive_dtype)) return FL_ERR_DTYPE;
  if (!sizes_ok(B, T, C) || !tensor_ok(gate, gate_dtype, gate_stride_b, gate_stride_t) ||
      !tensor_ok(drive, drive_dtype, drive_stride_b, drive_stride_t) || !tensor_ok(out, drive_dtype, 0, 0) ||
      !aligned(state_in, 4) || !aligned(state_out, 4) || !aligned(starts, 4))
    return FL_ERR_INVALID_ARGUMENT;
  if (!workspace_ok(workspace, workspace_bytes, fl_gated_scan_workspace_bytes(B, T, C, 0))) return FL_ERR_WORKSPACE;
  if (!aligned(workspace, 16)) return FL_ERR_INVALID_ARGUMENT;
  const Call c = call_of(gate, gate_stride_b, gate_stride_t, drive, drive_stride_b, drive_stride_t, B, T, C, workspace,
                         stream);
  const size_t bytes = word_bytes(B, T, C);
  FL_GATED(forward, c, bytes, state_in, state_out, starts, out)
}

int fl_gated_scan_backward(const void* gate, int gate_dtype, int per_token, int64_t gate_stride_b,
                           int64_t gate_stride_t, const void* drive, int drive_dtype, int64_t drive_stride_b,
                           int64_t drive_stride_t, int64_t B, int64_t T, int64_t C, const float* starts,
                           const void* g_out, const float* g_state, void* g_gate, void* g_drive, float* g_state_in,
                           void* workspace, size_t workspace_bytes, void* stream) {
  if (!dtype_ok(gate_dtype) || !dtype_ok(drive_dtype)) return FL_ERR_DTYPE;
  if (!sizes_ok(B, T, C) || !tensor_ok(gate, gate_dtype, gate_stride_b, gate_stride_t) ||
      !tensor_ok(drive, drive_dtype, drive_stride_b, drive_stride_t) || !aligned(g_gate, esize(gate_dtype)) ||
      !tensor_ok(g_drive, drive_dtype, 0, 0) || !aligned(g_out, esize(drive_dtype)) || !starts || !aligned(starts, 4) ||
      !aligned(g_state, 4) || !aligned(g_state_in, 4))
    return FL_ERR_INVALID_ARGUMENT;
  if (!workspace_ok(workspace, workspace_bytes, fl_gated_scan_workspace_bytes(B, T, C, 1))) return FL_ERR_WORKSPACE;
  if (!aligned(workspace, 16)) return FL_ERR_INVALID_ARGUMENT;
  const Call c = call_of(gate, gate_stride_b, gate_stride_t, drive, drive_stride_b, drive_stride_t, B, T, C, workspace,
                         stream);
  const size_t bytes = word_bytes(B, T, C);
  float* part = reinterpret_cast<float*>(static_cast<char*>(workspace) + bytes);
  FL_GATED(backward, c, bytes, starts, g_out, g_state, g_gate, g_drive, g_state_in, part)
}

#undef FL_GATED

}  // extern "C"
