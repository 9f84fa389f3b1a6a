// gated_scan.hip — the gated linear recurrence over T steps and its gradients:
//   h_t = a_t h_{t-1} + u_t,  h_{-1} = state_in or 0,          a gate to every channel or one to a token;
//   g_t = dh_t + a_{t+1} g_{t+1}  (the last step's carry is the final state's gradient),
//   du_t = g_t,  da_t = g_t h_{t-1} (summed over the channels where they share a gate),  dstate_in = a_0 g_0.
// The time is cut into tiles; a tile is a map h -> P h + S (P the product of its gates, S its end from 0), and maps
// compose. One launch forms the tiles' maps, one composes them, one runs every tile from its start.
#include "fl_common.h"

namespace {

using namespace fl;

constexpr int kTile = 256;  // steps
constexpr int64_t kMaxB = 65535, kMaxC = 64 * 65535, kMaxT = (int64_t)1 << 30;

struct Scan {
  const void* gate;
  const void* drive;
  int64_t gate_b, gate_t, drive_b, drive_t;  // strides in elements
  int64_t T, C, tiles;
  float2* maps;  // [B, tiles, C]
};

template <typename GT, bool TOKEN>
__device__ __forceinline__ float gate_at(const Scan& s, int64_t b, int64_t t, int64_t c) {
  return load_as<GT>(static_cast<const GT*>(s.gate) + b * s.gate_b + t * s.gate_t + (TOKEN ? 0 : c));
}
template <typename DT>
__device__ __forceinline__ float drive_at(const Scan& s, int64_t b, int64_t t, int64_t c) {
  return load_as<DT>(static_cast<const DT*>(s.drive) + b * s.drive_b + t * s.drive_t + c);
}

template <typename GT, typename DT, bool TOKEN>
__global__ __launch_bounds__(64) void fl_gated_map_kernel(const Scan s) {
  const int64_t b = blockIdx.z, tile = blockIdx.x, c = (int64_t)blockIdx.y * 64 + threadIdx.x;
  if (c >= s.C) return;
  const int64_t t0 = tile * kTile, t1 = t0 + kTile < s.T ? t0 + kTile : s.T;
  float p = 1.f, h = 0.f;
  for (int64_t t = t0; t < t1; ++t) {
    const float a = gate_at<GT, TOKEN>(s, b, t, c);
    h = fmaf(a, h, drive_at<DT>(s, b, t, c));
    p *= a;
  }
  s.maps[(b * s.tiles + tile) * s.C + c] = make_float2(p, h);
}

// the states that tiles start from
__global__ __launch_bounds__(64) void fl_gated_carry_kernel(const float2* __restrict__ maps, int64_t tiles, int64_t C,
                                                            const float* __restrict__ state_in,
                                                            float* __restrict__ starts, float* __restrict__ state_out) {
  const int64_t b = blockIdx.y, c = (int64_t)blockIdx.x * 64 + threadIdx.x;
  if (c >= C) return;
  float h = state_in ? state_in[b * C + c] : 0.f;
  for (int64_t i = 0; i < tiles; ++i) {
    const int64_t at = (b * tiles + i) * C + c;
    const float2 m = maps[at];
    starts[at] = h;
    h = fmaf(m.x, h, m.y);
  }
  if (state_out) state_out[b * C + c] = h;
}

template <typename GT, typename DT, bool TOKEN>
__global__ __launch_bounds__(64) void fl_gated_scan_kernel(const Scan s, const float* __restrict__ starts,
                                                           DT* __restrict__ out) {
  const int64_t b = blockIdx.z, tile = blockIdx.x, c = (int64_t)blockIdx.y * 64 + threadIdx.x;
  if (c >= s.C) return;
  const int64_t t0 = tile * kTile, t1 = t0 + kTile < s.T ? t0 + kTile : s.T;
  float h = starts[(b * s.tiles + tile) * s.C + c];
  for (int64_t t = t0; t < t1; ++t) {
    h = fmaf(gate_at<GT, TOKEN>(s, b, t, c), h, drive_at<DT>(s, b, t, c));
    store_as(out + (b * s.T + t) * s.C + c, h);
  }
}

// the reverse map of a tile: what its steps' gradients and the carry into its end make of the carry out of its start
template <typename GT, typename DT, bool TOKEN>
__global__ __launch_bounds__(64) void fl_gated_back_map_kernel(const Scan s, const DT* __restrict__ g_out) {
  const int64_t b = blockIdx.z, tile = blockIdx.x, c = (int64_t)blockIdx.y * 64 + threadIdx.x;
  if (c >= s.C) return;
  const int64_t t0 = tile * kTile, t1 = t0 + kTile < s.T ? t0 + kTile : s.T;
  float p = 1.f, k = 0.f;
  for (int64_t t = t1 - 1; t >= t0; --t) {
    const float a = gate_at<GT, TOKEN>(s, b, t, c);
    k = a * (k + (g_out ? load_as<DT>(g_out + (b * s.T + t) * s.C + c) : 0.f));
    p *= a;
  }
  s.maps[(b * s.tiles + tile) * s.C + c] = make_float2(p, k);
}

__global__ __launch_bounds__(64) void fl_gated_back_carry_kernel(float2* __restrict__ maps, int64_t tiles, int64_t C,
                                                                 const float* __restrict__ g_state,
                                                                 float* __restrict__ g_state_in) {
  const int64_t b = blockIdx.y, c = (int64_t)blockIdx.x * 64 + threadIdx.x;
  if (c >= C) return;
  float k = g_state ? g_state[b * C + c] : 0.f;
  for (int64_t i = tiles - 1; i >= 0; --i) {
    const int64_t at = (b * tiles + i) * C + c;
    const float2 m = maps[at];
    maps[at].x = k;  // the carry into the tile's end
    k = fmaf(m.x, k, m.y);
  }
  if (g_state_in) g_state_in[b * C + c] = k;
}

// A tile's states again, kept in the LDS, then its steps from the last to the first.
template <typename GT, typename DT, bool TOKEN>
__global__ __launch_bounds__(64) void fl_gated_back_kernel(const Scan s, const float* __restrict__ starts,
                                                           const DT* __restrict__ g_out, GT* __restrict__ g_gate,
                                                           float* __restrict__ part, DT* __restrict__ g_drive) {
  __shared__ float s_h[kTile][64];
  const int lane = threadIdx.x;
  const int64_t b = blockIdx.z, tile = blockIdx.x, c = (int64_t)blockIdx.y * 64 + lane;
  const bool ok = c < s.C;
  const int64_t cc = ok ? c : s.C - 1;
  const int64_t t0 = tile * kTile, t1 = t0 + kTile < s.T ? t0 + kTile : s.T;
  float h = starts[(b * s.tiles + tile) * s.C + cc];
  for (int64_t t = t0; t < t1; ++t) {
    s_h[t - t0][lane] = h;  // the state before the step
    h = fmaf(gate_at<GT, TOKEN>(s, b, t, cc), h, drive_at<DT>(s, b, t, cc));
  }
  float k = s.maps[(b * s.tiles + tile) * s.C + cc].x;
  for (int64_t t = t1 - 1; t >= t0; --t) {
    const int64_t at = (b * s.T + t) * s.C + cc;
    const float g = (g_out ? load_as<DT>(g_out + at) : 0.f) + k;
    const float da = g * s_h[t - t0][lane];
    if (ok) store_as(g_drive + at, g);
    if (!g_gate) {
    } else if constexpr (TOKEN) {
      const float sum = wave_sum(ok ? da : 0.f);
      if (lane == 0) part[((int64_t)blockIdx.y * gridDim.z + b) * s.T + t] = sum;
    } else {
      if (ok) store_as(g_gate + at, da);
    }
    k = gate_at<GT, TOKEN>(s, b, t, cc) * g;
  }
}

// the gradient of a token's gate: the sums of its groups of channels, in their order
template <typename GT>
__global__ __launch_bounds__(256) void fl_gated_token_kernel(const float* __restrict__ part, int64_t n, int64_t groups,
                                                             GT* __restrict__ g_gate) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  float sum = 0.f;
  for (int64_t k = 0; k < groups; ++k) sum += part[k * n + i];
  store_as(g_gate + i, sum);
}

struct Call {
  Scan s;
  int64_t B;
  hipStream_t stream;
  dim3 tiles() const { return dim3((unsigned)s.tiles, (unsigned)cdiv(s.C, 64), (unsigned)B); }
  dim3 chains() const { return dim3((unsigned)cdiv(s.C, 64), (unsigned)B); }
};

template <typename GT, typename DT, bool TOKEN>
int forward(const Call& c, const float* state_in, float* state_out, float* starts, void* out) {
  fl_gated_map_kernel<GT, DT, TOKEN><<<c.tiles(), 64, 0, c.stream>>>(c.s);
  fl_gated_carry_kernel<<<c.chains(), 64, 0, c.stream>>>(c.s.maps, c.s.tiles, c.s.C, state_in, starts, state_out);
  fl_gated_scan_kernel<GT, DT, TOKEN><<<c.tiles(), 64, 0, c.stream>>>(c.s, starts, static_cast<DT*>(out));
  return hip_status(hipGetLastError());
}

template <typename GT, typename DT, bool TOKEN>
int backward(const Call& c, const float* starts, const void* g_out, const float* g_state, void* g_gate, void* g_drive,
             float* g_state_in, float* part) {
  const DT* g = static_cast<const DT*>(g_out);
  fl_gated_back_map_kernel<GT, DT, TOKEN><<<c.tiles(), 64, 0, c.stream>>>(c.s, g);
  fl_gated_back_carry_kernel<<<c.chains(), 64, 0, c.stream>>>(c.s.maps, c.s.tiles, c.s.C, g_state, g_state_in);
  fl_gated_back_kernel<GT, DT, TOKEN><<<c.tiles(), 64, 0, c.stream>>>(c.s, starts, g, static_cast<GT*>(g_gate), part,
                                                                       static_cast<DT*>(g_drive));
  if (TOKEN && g_gate) {
    const int64_t n = c.B * c.s.T;
    fl_gated_token_kernel<GT><<<(unsigned)cdiv(n, 256), 256, 0, c.stream>>>(part, n, cdiv(c.s.C, 64),
                                                                            static_cast<GT*>(g_gate));
  }
  return hip_status(hipGetLastError());
}

bool sizes_ok(int64_t B, int64_t T, int64_t C) {
  return B > 0 && T > 0 && C > 0 && B <= kMaxB && C <= kMaxC && T <= kMaxT;
}

bool tensor_ok(const void* p, int dtype, int64_t stride_b, int64_t stride_t) {
  return p && aligned(p, esize(dtype)) && stride_b >= 0 && stride_t >= 0;
}

}  // namespace

extern "C" {

int64_t fl_gated_scan_tile(void) { return kTile; }

size_t fl_gated_scan_workspace_bytes(int64_t B, int64_t T, int64_t C, int backward) {
  if (!sizes_ok(B, T, C)) return 0;
  return (size_t)(B * cdiv(T, kTile) * C) * 8 + (size_t)(B * cdiv(T, kTile) * C) * 4 +
         (backward ? (size_t)(cdiv(C, 64) * B * T) * 4 : 0);
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
  if (!workspace || workspace_bytes < fl_gated_scan_workspace_bytes(B, T, C, 0)) return FL_ERR_WORKSPACE;
  if (!aligned(workspace, 16)) return FL_ERR_INVALID_ARGUMENT;
  const int64_t tiles = cdiv(T, kTile);
  float2* maps = static_cast<float2*>(workspace);
  if (!starts) starts = reinterpret_cast<float*>(maps + B * tiles * C);
  const Call c{{gate, drive, gate_stride_b, gate_stride_t, drive_stride_b, drive_stride_t, T, C, tiles, maps}, B,
               static_cast<hipStream_t>(stream)};
  FL_GATED(forward, c, state_in, state_out, starts, out)
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
  if (!workspace || workspace_bytes < fl_gated_scan_workspace_bytes(B, T, C, 1)) return FL_ERR_WORKSPACE;
  if (!aligned(workspace, 16)) return FL_ERR_INVALID_ARGUMENT;
  const int64_t tiles = cdiv(T, kTile);
  float2* maps = static_cast<float2*>(workspace);
  float* part = reinterpret_cast<float*>(maps + B * tiles * C);
  const Call c{{gate, drive, gate_stride_b, gate_stride_t, drive_stride_b, drive_stride_t, T, C, tiles, maps}, B,
               static_cast<hipStream_t>(stream)};
  FL_GATED(backward, c, starts, g_out, g_state, g_gate, g_drive, g_state_in, part)
}

#undef FL_GATED

}  // extern "C"
