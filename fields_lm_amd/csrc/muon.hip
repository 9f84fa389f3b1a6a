// muon.hip — matrices brought near their closest semi-orthogonal ones by Newton-Schulz steps, on their own and in a Muon
// step over many matrices at once.
//
//   X = G / (|G|_F + eps), then `steps` times X <- a X + (b A + c A^2) X with A = X X^T.
//
// A tall matrix is taken transposed, so that X is m x n with m <= n. The steps run on the m x m side: with
// P = a I + b A + c A^2 a step is X <- P X and makes A into P A P, and all of these commute and are symmetric. So k steps
// are one product X X^T, products of symmetric matrices (of which the lower half is computed) and one product
// (P_k .. P_1) X. A's small eigenvalues are squares of X's singular values, and a step lets their error grow a^2-fold
// (12 for the usual a) where X's own grows a-fold: after at most kStage steps, one where sums are short, X is formed and A
// taken from it anew, which keeps results as near to the formula's as steps on X in fp32 are.
//
// Every matrix is held as two fp16 planes, high and low part of its values times a power of two (22 bits), and a product
// is three of matrix instructions, high high + high low + low high, summed in fp32: bf16 operands end 3% from the result
// where singular values are alike, and as far as it is long where a few are strong.
//
// Bound by the operands, past the L2: 64 squares of 1,024 x 1,024 take 157 to 165 us a product (1.4 to 1.5 PFLOP/s of fp16, of
// which a third counts; registers alone reach 1.7 on such values), and 110 matrices of a model, 0.27 G values, 14.7 ms
// (steps on X in fp32 library products 80), in which matrix instructions hold their units for 41 to 55% of the cycles in which a
// CU has work: a product with X moves 10.6 GB in 2.1 ms (5.0 TB/s), five times its operands, the others move 2.8 to 4.3
// TB/s. A single 256 x 632 matrix, 20 dependent launches, takes 123 us (1,175). What was tried and is no faster (110 matrices, 15.9 ms at the time): tiles of 256 x 256 (15.2
// to 19.0), 256 x 128 with three buffers (18.3), 128 x 128 with four and one block to a CU (17.8), all of a step's reads
// ahead of its products (17.2), wave priority (1% slower), waves above the diagonal left idle (4% slower).
#include "fl_common.h"

#include <math.h>

#include <algorithm>
#include <type_traits>
#include <vector>

namespace {

using namespace fl;

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 half_t;

constexpr int kStage = 3;      // steps between two products with X at most, where one
                               // does not have to do:
constexpr int64_t kLongSide = 256;  // where the short side is this long, or results are bf16
constexpr int kPad = 32;       // rows of planes are a multiple of this long, zeros behind the matrix
constexpr int kSquares = 5;    // m x m matrices of the workspace
constexpr int kCopyTile = 64;  // of the tile that is laid out by a block
constexpr int kTable = 56;     // matrices to a launch that sets up their table
constexpr int kNormChunk = 4096;  // values of a block of the norm (one matrix of 256 x 632: 3.6 us, 12 with 16,384 values read one by one)
constexpr int64_t kMaxMatrices = 1 << 20, kMaxSide = 1 << 20, kMaxValues = (int64_t)1 << 30;
constexpr int kFold = 16;      // steps of 32 columns
constexpr int kTile = 128, kSmallTile = 64;  // rows and columns of a product's tile
constexpr int64_t kSlots = 512, kIdle = 150;  // tiles that run at a time (two to a CU)
// (110 matrices of a model: groups of 1 GiB 15.3 ms, 2 GiB 14.7, 4 GiB 14.6)
constexpr size_t kGroupBytes = (size_t)2 << 30;  // matrices are taken in groups of at most about this much workspace
constexpr int kMaxSteps = 64;
constexpr double kMaxBound = 1024.0;  // of singular values

struct Mat {
  half_t* base;    // X [m, ldn], X^T [n, ldm] twice, squares [m, ldm], 2 ld halves to a row: 32 high parts, their low ones
  const void* g;
  float* buf;
  void* p;
  int m, n;        // m <= n
  int tall;        // g and p are n x m
  float lr_scale;
  int first_norm, first_copy, first_square, first_apply;  // running counts of blocks
};

struct Table {
  Mat mat[kTable];
  int n;
};

__host__ __device__ __forceinline__ int64_t padded(int64_t x) { return (x + kPad - 1) / kPad * kPad; }

__global__ __launch_bounds__(64) void fl_muon_table_kernel(const Table t, Mat* __restrict__ out) {
  if ((int)threadIdx.x < t.n) out[threadIdx.x] = t.mat[threadIdx.x];
}

// the matrix whose blocks, counted by FIRST, hold `block`: the last that begins at or before it, 64 of them tried at
// a time (4,096 matrices of 64 x 64 1.5 ms, 3.9 by counting all that begin before it)
template <int Mat::*FIRST>
__device__ __forceinline__ int matrix_of(const Mat* mats, int n, int block) {
  const int lane = threadIdx.x & 63;
  int at = 0;
  for (int left = n; left > 1;) {
    const int step = (left + 63) / 64, k = lane * step;
    const int last = __popcll(__ballot(k < left && mats[at + min(k, left - 1)].*FIRST <= block)) - 1;
    at += last * step;
    left = min(step, left - last * step);
  }
  return uniform(at);
}

struct Update {
  int is_bf16;   // g, p
  int muon;      // 0: orthogonalize, g the matrix and p the result
  float mu, keep;  // momentum and 1 - momentum
  int nesterov;
  const float* grad_scale;
  const float* lr_ptr;
  float lr, decay;
};

__device__ __forceinline__ float load_any(const void* p, int64_t i, int is_bf16) {
  return is_bf16 ? load_as<bf16_bits>(static_cast<const bf16_bits*>(p) + i) : static_cast<const float*>(p)[i];
}

__device__ __forceinline__ bool skipped(const Update& u) {
  return u.grad_scale && !(fabsf(*u.grad_scale) <= 3.4028235e38f);
}

// four values at any element's address
__device__ __forceinline__ f32x4 load4(const void* p, int64_t i, int is_bf16) {
  f32x4 v;
  if (is_bf16) {
    const u32x2 r = *reinterpret_cast<const u32x2_any*>(static_cast<const bf16_bits*>(p) + i);
    v = f32x4{bf16_lo(r[0]), bf16_hi(r[0]), bf16_lo(r[1]), bf16_hi(r[1])};
  } else {
    const u32x4 r = *reinterpret_cast<const u32x4_any*>(static_cast<const float*>(p) + i);
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = __uint_as_float(r[k]);
  }
  return v;
}

// The momentum's update (Muon) and the sum of the squares of what is orthogonalized, in fp64.
__global__ __launch_bounds__(256) void fl_muon_norm_kernel(const Mat* __restrict__ mats, int n, const Update u,
                                                           double* __restrict__ part) {
  __shared__ double s_sum[4];
  const int i = matrix_of<&Mat::first_norm>(mats, n, blockIdx.x);
  const Mat& k = mats[i];
  const int64_t numel = (int64_t)k.m * k.n, lo = (int64_t)((int)blockIdx.x - k.first_norm) * kNormChunk;
  const float scale = u.grad_scale ? *u.grad_scale : 1.f;
  const bool skip = skipped(u);
  double sum = 0.0;
  const auto one = [&](float v, float& b) {  // what is orthogonalized of a value, its buffer brought forward
    if (u.muon) {
      v *= scale;
      b = fmaf(u.mu, b, u.keep * v);
      v = u.nesterov ? fmaf(u.keep, v, u.mu * b) : b;
    }
    sum = fma((double)v, (double)v, sum);
  };
  constexpr int kPacks = kNormChunk / 1024;
  if (lo + kNormChunk <= numel) {
    f32x4 v[kPacks], b[kPacks];
#pragma unroll
    for (int j = 0; j < kPacks; ++j) {
      const int64_t at = lo + j * 1024 + threadIdx.x * 4;
      v[j] = load4(k.g, at, u.is_bf16);
      if (u.muon) b[j] = load4(k.buf, at, 0);
    }
#pragma unroll
    for (int j = 0; j < kPacks; ++j) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        float x = b[j][q];
        one(v[j][q], x);
        b[j][q] = x;
      }
      if (u.muon && !skip) {
        u32x4 r;
#pragma unroll
        for (int q = 0; q < 4; ++q) r[q] = __float_as_uint(b[j][q]);
        *reinterpret_cast<u32x4_any*>(k.buf + lo + j * 1024 + threadIdx.x * 4) = r;
      }
    }
  } else {
    for (int64_t j = lo + threadIdx.x; j < numel; j += 256) {
      float b = u.muon ? k.buf[j] : 0.f;
      one(load_any(k.g, j, u.is_bf16), b);
      if (u.muon && !skip) k.buf[j] = b;
    }
  }
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) sum += __shfl_xor(sum, d);
  if ((threadIdx.x & 63) == 0) s_sum[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) part[blockIdx.x] = (s_sum[0] + s_sum[1]) + (s_sum[2] + s_sum[3]);
}

// high and low part of v, in bits 15..0 and 31..16
__device__ __forceinline__ uint32_t split(float v) {
  const half_t hi = (half_t)v, lo = (half_t)(v - (float)hi);
  return (uint32_t)__builtin_bit_cast(unsigned short, hi) | (uint32_t)__builtin_bit_cast(unsigned short, lo) << 16;
}
// where a row of halves has the high part of column c; its low part is kPad further on
__device__ __forceinline__ int64_t column(int64_t c) { return (c >> 5) * 64 + (c & 31); }
// the high (or low) parts of two values
__device__ __forceinline__ uint32_t highs(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x05040100); }
__device__ __forceinline__ uint32_t lows(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x07060302); }

// X = G / (|G| + eps) times x_scale, as planes of X and of X^T, a tile of 64 x 64 to a block.
__global__ __launch_bounds__(256) void fl_muon_copy_kernel(const Mat* __restrict__ mats, int n, const Update u,
                                                           const double* __restrict__ part, double eps, float x_scale) {
  __shared__ uint32_t s_x[kCopyTile][kCopyTile + 1];
  __shared__ double s_sum[4];
  const int i = matrix_of<&Mat::first_copy>(mats, n, blockIdx.x);
  const Mat& k = mats[i];
  const int64_t numel = (int64_t)k.m * k.n;
  double sum = 0.0;
  const int64_t blocks = (numel + kNormChunk - 1) / kNormChunk;
  for (int64_t j = threadIdx.x; j < blocks; j += 256) sum += part[k.first_norm + j];
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) sum += __shfl_xor(sum, d);
  if ((threadIdx.x & 63) == 0) s_sum[threadIdx.x >> 6] = sum;
  __syncthreads();
  sum = (s_sum[0] + s_sum[1]) + (s_sum[2] + s_sum[3]);
  const double inv = sum == 0.0 ? 0.0 : (double)x_scale / (sqrt(sum) + eps);  // (zeros stay zeros, whatever eps is)

  // the matrix as it lies: rows x cols
  const int rows = k.tall ? k.n : k.m, cols = k.tall ? k.m : k.n;
  const int64_t ld_r = padded(cols), ld_c = padded(rows);
  half_t* x = k.base;
  half_t* xt = x + 2 * (int64_t)k.m * padded(k.n);
  half_t* straight = k.tall ? xt : x;   // rows as they lie
  half_t* turned = k.tall ? x : xt;
  const int across = (int)((ld_r + kCopyTile - 1) / kCopyTile), tile = (int)blockIdx.x - k.first_copy;
  const int r0 = tile / across * kCopyTile, c0 = tile % across * kCopyTile;
  const float scale = u.grad_scale ? *u.grad_scale : 1.f;
  const auto value = [&](float g, float b) {
    if (u.muon) g = u.nesterov ? fmaf(u.keep, g * scale, u.mu * b) : b;
    return split((float)((double)g * inv));
  };
#pragma unroll
  for (int j = 0; j < kCopyTile * kCopyTile / 1024; ++j) {
    const int rr = j * 16 + (threadIdx.x >> 4), cc = (threadIdx.x & 15) * 4, r = r0 + rr, c = c0 + cc;
    const int64_t at = (int64_t)r * cols + c;
    u32x4 w = {0, 0, 0, 0};
    if (r < rows && c + 4 <= cols) {
      const f32x4 g = u.muon && !u.nesterov ? f32x4{0.f, 0.f, 0.f, 0.f} : load4(k.g, at, u.is_bf16);
      const f32x4 b = u.muon ? load4(k.buf, at, 0) : g;
#pragma unroll
      for (int q = 0; q < 4; ++q) w[q] = value(g[q], b[q]);
    } else if (r < rows) {
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (c + q < cols) w[q] = value(load_any(k.g, at + q, u.is_bf16), u.muon ? k.buf[at + q] : 0.f);
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) s_x[rr][cc + q] = w[q];
  }
  __syncthreads();
  // 32 columns of a row to a line of 128 bytes: its high and low parts, eight lanes with 16 bytes each
  for (int j = threadIdx.x; j < kCopyTile * 2 * 8; j += 256) {
    const int line = j >> 3, part = j & 7, i = line >> 1, half = line & 1, from = half * 32 + (part & 3) * 8;
    u32x4 v;
    if (r0 + i < rows && c0 + half * 32 < ld_r) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const uint32_t x0 = s_x[i][from + 2 * q], x1 = s_x[i][from + 2 * q + 1];
        v[q] = part < 4 ? highs(x0, x1) : lows(x0, x1);
      }
      *reinterpret_cast<u32x4*>(straight + (int64_t)(r0 + i) * 2 * ld_r + (c0 / 32 + half) * 64 + part * 8) = v;
    }
    if (c0 + i < cols && r0 + half * 32 < ld_c) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const uint32_t x0 = s_x[from + 2 * q][i], x1 = s_x[from + 2 * q + 1][i];
        v[q] = part < 4 ? highs(x0, x1) : lows(x0, x1);
      }
      *reinterpret_cast<u32x4*>(turned + (int64_t)(c0 + i) * 2 * ld_c + (r0 / 32 + half) * 64 + part * 8) = v;
    }
  }
}

// What a product is formed of: L R^T of rows of X, of X^T or of a square.
struct Product {
  int left[2], right[2], out[2];  // squares' numbers, for up to two products of a launch
  float norm[2], out_scale[2];    // 1 / (the operands' scales); the result's
  float a, b, c, in_scale;        // of the polynomial, and 1 / the scale of the square that it reads
  int source;                     // which X^T
};

enum Kind { kGram, kPoly, kSquare, kApply, kFinal };

// 16 values of a parameter, `left` of them there: p keep - rate v, or v itself
template <typename T>
__device__ __forceinline__ void update16(T* p, int left, const float* v, int muon, float keep, float rate) {
  if (left >= 16) {
    constexpr int N = 16 / sizeof(T);
    u32x4_any* to = reinterpret_cast<u32x4_any*>(p);
    u32x4 old[16 / N];
#pragma unroll
    for (int i = 0; i < 16 / N; ++i) old[i] = muon ? (u32x4)to[i] : u32x4{0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 16 / N; ++i) {
      u32x4 r;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if constexpr (N == 4) {
          const float x = v[4 * i + k];
          r[k] = __float_as_uint(muon ? fmaf(-rate, x, __uint_as_float(old[i][k]) * keep) : x);
        } else {
          const float x = v[8 * i + 2 * k], y = v[8 * i + 2 * k + 1];
          r[k] = muon ? bf16_pair(fmaf(-rate, x, bf16_lo(old[i][k]) * keep), fmaf(-rate, y, bf16_hi(old[i][k]) * keep))
                      : bf16_pair(x, y);
        }
      }
      to[i] = r;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (i < left) store_as(p + i, muon ? fmaf(-rate, v[i], load_as<T>(p + i) * keep) : v[i]);
  }
}

// A tile's sizes: TILE rows and columns by WR x WC waves, and how many steps of 32 columns a buffer of the LDS holds.
template <int TILE>
struct Shape;
template <>
struct Shape<kTile> {
  static constexpr int WR = 2, WC = 2, BATCH = 1;
};
template <>
struct Shape<kSmallTile> {
  static constexpr int WR = 2, WC = 2, BATCH = 4;
};
template <int TILE>
constexpr int threads_of() { return Shape<TILE>::WR * Shape<TILE>::WC * 64; }

// The blocks of a launch come to the card's eight dies in turn, so that runs of kRun tiles, which read the same rows, are
// given to one of them.
constexpr int kRun = 16;
__device__ __forceinline__ int tile_of(int block) {
  const int die = block & 7, i = block >> 3;
  return (i / kRun * 8 + die) * kRun + i % kRun;
}

// One tile of L R^T. Rows past an operand's last are read as its last one; what they give is not written.
// The LDS holds two buffers: while one is multiplied the next is loaded straight into the other. 32 columns of a row are a
// line of 128 bytes, high parts before low ones, whose eight packs change places by half the row's number, so that sixteen
// rows' equal packs lie in different banks of the 64.
template <int KIND, int TILE>
__global__ __launch_bounds__(threads_of<TILE>(), TILE == kTile ? 2 : 1) void fl_muon_product_kernel(const Mat* __restrict__ mats, int n,
                                                                             int tiles, const Product q,
                                                                             const Update u) {
  constexpr bool kSymmetric = KIND <= kSquare;
  constexpr int WR = Shape<TILE>::WR, WC = Shape<TILE>::WC, BATCH = Shape<TILE>::BATCH, kWaves = WR * WC;
  constexpr int NI = TILE / WR / 32, NJ = TILE / WC / 32;
  constexpr int kLine = 128, kStepBytes = TILE * kLine, kOperand = BATCH * kStepBytes, kBuffer = 2 * kOperand;
  constexpr int kTurn = 36;  // words of a row of the tile that is turned in the LDS
  static_assert(kWaves * 32 * kTurn * 4 <= 2 * kBuffer, "");
  __shared__ __attribute__((aligned(128))) char s_tile[2 * kBuffer];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int job = blockIdx.y, index = tile_of((int)blockIdx.x);
  if (index >= tiles) return;
  const int which = kSymmetric ? matrix_of<&Mat::first_square>(mats, n, index)
                               : matrix_of<&Mat::first_apply>(mats, n, index);
  const Mat& k = mats[which];
  const int m = k.m, cols = k.n;
  const int64_t ldn = padded(cols), ldm = padded(m);
  half_t* x = k.base;
  half_t* xt[2] = {x + 2 * (int64_t)m * ldn, x + 2 * (int64_t)m * ldn + 2 * cols * ldm};
  half_t* squares = xt[1] + 2 * cols * ldm;
  const int64_t square = 2 * (int64_t)m * ldm;

  // operands: rows, their count, their length
  const half_t *lp, *rp;
  int l_rows, r_rows, ti, tj;
  int64_t ld;
  const bool turn = KIND == kFinal && k.tall;
  if constexpr (kSymmetric) {
    const int t = index - k.first_square;
    ti = (int)((sqrtf(8.f * t + 1.f) - 1.f) * 0.5f);
    while (ti * (ti + 1) / 2 > t) --ti;
    while ((ti + 1) * (ti + 2) / 2 <= t) ++ti;
    tj = t - ti * (ti + 1) / 2;
    l_rows = r_rows = m;
    if constexpr (KIND == kGram) {
      lp = rp = x;
      ld = ldn;
    } else {
      lp = squares + q.left[job] * square;
      rp = squares + q.right[job] * square;
      ld = ldm;
    }
  } else {
    const half_t* sq = squares + q.left[0] * square;
    lp = turn ? xt[q.source] : sq;
    rp = turn ? sq : xt[q.source];
    l_rows = turn ? cols : m;
    r_rows = turn ? m : cols;
    ld = ldm;
    const int across = (r_rows + TILE - 1) / TILE, t = index - k.first_apply;
    ti = t / across;
    tj = t - ti * across;
  }
  ti = uniform(ti);
  tj = uniform(tj);
  const int r0 = ti * TILE, c0 = tj * TILE;
  const int steps = (int)(ld / 32);

  // eight lines to an instruction
  const int load_row = lane >> 3;
  auto load = [&](int buffer, int step) {
    constexpr int kPieces = TILE / 8 / kWaves;  // of an operand's step, to a wave
#pragma unroll
    for (int b = 0; b < BATCH; ++b) {
      if (BATCH > 1 && step + b >= steps) break;
#pragma unroll
      for (int o = 0; o < 2; ++o) {
        const half_t* base = o ? rp : lp;
        const int rows = o ? r_rows : l_rows, first = o ? c0 : r0;
#pragma unroll
        for (int j = 0; j < kPieces; ++j) {
          const int rr = (wave * kPieces + j) * 8;
          const int row = min(first + rr + load_row, rows - 1);
          const int pack = (lane & 7) ^ (((rr + load_row) >> 1) & 7);
          const half_t* from = base + row * 2 * ld + (step + b) * 64 + pack * 8;
          __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from,
                                           (__attribute__((address_space(3))) void*)(s_tile + buffer * kBuffer +
                                                                                     o * kOperand + b * kStepBytes +
                                                                                     rr * kLine),
                                           16, 0, 0);
        }
      }
    }
  };

  const int wr = wave / WC * (TILE / WR), wc = wave % WC * (TILE / WC);
  const f32x16 none = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  f32x16 acc[NI][NJ], part[NI][NJ];
#pragma unroll
  for (int i = 0; i < NI; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j) acc[i][j] = part[i][j] = none;

  const char* l_at = s_tile + (wr + (lane & 31)) * kLine;
  const char* r_at = s_tile + kOperand + (wc + (lane & 31)) * kLine;
  // Sums: 512 columns at a time, which a second sum takes (a wide matrix's 1,286 columns in one: 3 times the error). While
  // that is empty it holds the products with low parts, which are 2^-11 of the others and round nothing of them off.
  const auto multiply = [&](int at, auto first) {
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      f16x8 l[NI][2], r[NJ][2];
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const int pack = ((p * 4 + kk * 2 + (lane >> 5)) ^ ((lane >> 1) & 7)) * 16 + at;
#pragma unroll
        for (int j = 0; j < NJ; ++j) r[j][p] = *reinterpret_cast<const f16x8*>(r_at + j * 32 * kLine + pack);
#pragma unroll
        for (int i = 0; i < NI; ++i) l[i][p] = *reinterpret_cast<const f16x8*>(l_at + i * 32 * kLine + pack);
      }
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          f32x16& low = decltype(first)::value ? acc[i][j] : part[i][j];
          part[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(l[i][0], r[j][0], part[i][j], 0, 0, 0);
          low = __builtin_amdgcn_mfma_f32_32x32x16_f16(l[i][0], r[j][1], low, 0, 0, 0);
          low = __builtin_amdgcn_mfma_f32_32x32x16_f16(l[i][1], r[j][0], low, 0, 0, 0);
        }
    }
  };
  const auto fold = [&] {
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        acc[i][j] += part[i][j];
        part[i][j] = none;
      }
  };
  load(0, 0);
  int buffer = 0, s = 0;
  const auto sum = [&](int end, auto first) {
    for (; s < end; s += BATCH, buffer ^= 1) {
      __builtin_amdgcn_s_waitcnt(0);
      __syncthreads();  // the buffer is there, and nobody reads the other one any more
      if (s + BATCH < steps) load(buffer ^ 1, s + BATCH);
#pragma unroll
      for (int b = 0; b < BATCH; ++b) {
        if (BATCH > 1 && s + b >= steps) break;
        multiply(buffer * kBuffer + b * kStepBytes, first);
      }
    }
    fold();
  };
  sum(min(steps, kFold), std::true_type());
  while (s < steps) sum(min(steps, s + kFold), std::false_type());

  if constexpr (KIND == kFinal) {
    const float lr = u.muon ? (u.lr_ptr ? *u.lr_ptr : u.lr) : 0.f;
    const float keep = 1.f - lr * u.decay, rate = lr * k.lr_scale;
    if (u.muon && skipped(u)) return;
    float* s_turn = reinterpret_cast<float*>(s_tile) + wave * 32 * kTurn;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const int rb = r0 + wr + i * 32, cb = c0 + wc + j * 32;
        if (rb >= l_rows || cb >= r_rows) continue;  // (the same in the whole wave)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          s_turn[(8 * (e >> 2) + 4 * (lane >> 5) + (e & 3)) * kTurn + (lane & 31)] = acc[i][j][e] * q.norm[0];
        __builtin_amdgcn_wave_barrier();
        const int row = rb + (lane >> 1), col = cb + (lane & 1) * 16;
        float v[16];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const f32x4 w = *reinterpret_cast<const f32x4*>(s_turn + (lane >> 1) * kTurn + (lane & 1) * 16 + 4 * e);
#pragma unroll
          for (int f = 0; f < 4; ++f) v[4 * e + f] = w[f];
        }
        __builtin_amdgcn_wave_barrier();
        if (row >= l_rows) continue;
        const int64_t at = (int64_t)row * r_rows + col;
        if (u.is_bf16)
          update16(static_cast<bf16_bits*>(k.p) + at, r_rows - col, v, u.muon, keep, rate);
        else
          update16(static_cast<float*>(k.p) + at, r_rows - col, v, u.muon, keep, rate);
      }
  } else {
    // `straight` has the tile's rows, `turned` its columns; both get the zeros behind their rows. Of a square what
    // is below the diagonal stands for what is above (which may differ in its last bits), so that no tile's size shows.
    const int rows = m, columns = kSymmetric ? m : cols;
    const int64_t ld_c = kSymmetric ? ldm : ldn, ld_r = ldm;
    half_t* straight = kSymmetric ? squares + q.out[job] * square : x;
    half_t* turned = kSymmetric ? straight : xt[1 - q.source];
    const float norm = q.norm[job], out_scale = q.out_scale[job];
    const half_t* poly = squares + q.left[job] * square;
    uint32_t* s_turn = reinterpret_cast<uint32_t*>(s_tile) + wave * 32 * kTurn;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const int rb = r0 + wr + i * 32, cb = c0 + wc + j * 32, col = cb + (lane & 31);
        if (rb >= ld_r || cb >= ld_c || (kSymmetric && rb < cb)) continue;  // (the same in the whole wave)
        const bool diagonal = kSymmetric && rb == cb;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int row = rb + 8 * g + 4 * (lane >> 5);
          f16x4 hi = {0, 0, 0, 0}, lo = {0, 0, 0, 0};
          if constexpr (KIND == kPoly) {  // the square's own values, read as those across the diagonal
            const half_t* from = poly + (int64_t)min(col, m - 1) * 2 * ldm + column(row);
            hi = *reinterpret_cast<const f16x4*>(from);
            lo = *reinterpret_cast<const f16x4*>(from + kPad);
          }
          u32x4 w;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float v = acc[i][j][4 * g + e] * norm;
            if constexpr (KIND == kPoly)
              v = q.b * ((float)hi[e] + (float)lo[e]) * q.in_scale + q.c * v + (row + e == col ? q.a : 0.f);
            w[e] = split(row + e < rows && col < columns ? v * out_scale : 0.f);
          }
          if (!diagonal && col < columns) {
            half_t* to = turned + (int64_t)col * 2 * ld_r + column(row);
            *reinterpret_cast<u32x2*>(to) = u32x2{highs(w[0], w[1]), highs(w[2], w[3])};
            *reinterpret_cast<u32x2*>(to + kPad) = u32x2{lows(w[0], w[1]), lows(w[2], w[3])};
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) s_turn[(8 * g + 4 * (lane >> 5) + e) * kTurn + (lane & 31)] = w[e];
        }
        // (a wave's own part of the LDS: its reads come behind its writes)
        __builtin_amdgcn_wave_barrier();
        const int row = rb + (lane >> 1), half = (lane & 1) * 16;
        u32x4 w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          w[e] = *reinterpret_cast<const u32x4*>(s_turn + (lane >> 1) * kTurn + half + 4 * e);
        if (diagonal) {
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (half + e > lane >> 1) w[e >> 2][e & 3] = s_turn[(half + e) * kTurn + (lane >> 1)];
        }
        __builtin_amdgcn_wave_barrier();
        if (row < rows) {
          half_t* to = straight + (int64_t)row * 2 * ld_c + column(cb) + half;
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const u32x4 p = w[2 * e], o = w[2 * e + 1];
            *reinterpret_cast<u32x4*>(to + 8 * e) =
                u32x4{highs(p[0], p[1]), highs(p[2], p[3]), highs(o[0], o[1]), highs(o[2], o[3])};
            *reinterpret_cast<u32x4*>(to + kPad + 8 * e) =
                u32x4{lows(p[0], p[1]), lows(p[2], p[3]), lows(o[0], o[1]), lows(o[2], o[3])};
          }
        }
      }
  }
}

// ---------------------------------------------------------------- host

size_t planes_bytes(int64_t rows, int64_t cols) {
  const int64_t m = rows < cols ? rows : cols, n = rows < cols ? cols : rows;
  return (size_t)(2 * m * padded(n) + 4 * n * padded(m) + kSquares * 2 * m * padded(m)) * sizeof(half_t);
}

int64_t norm_blocks(int64_t rows, int64_t cols) { return cdiv(rows * cols, kNormChunk); }

bool lists_ok(int64_t n, const int64_t* rows, const int64_t* cols) {
  if (n <= 0 || n > kMaxMatrices || !rows || !cols) return false;
  for (int64_t i = 0; i < n; ++i)
    if (rows[i] < 0 || cols[i] < 0 || rows[i] > kMaxSide || cols[i] > kMaxSide || rows[i] * cols[i] > kMaxValues)
      return false;
  return true;
}

// The group of matrices from i on: where it ends, and its planes', sums' and table's bytes.
struct Group {
  int64_t end, count, sums;
  size_t planes;
  size_t bytes() const { return planes + (size_t)sums * 8 + (size_t)count * sizeof(Mat); }
};

// lower half of an m x m square in tiles
int64_t square_tiles(int64_t m, int tile) {
  const int64_t side = cdiv(m, tile);
  return side * (side + 1) / 2;
}

// What a group's product of squares takes, in tiles of a card that runs kSlots at a time, a launch's start and end counted
// as kIdle.
int64_t cost(int64_t tiles) { return tiles ? cdiv(tiles, kSlots) * kSlots + kIdle : 0; }

// Stages of one step lose nothing on steps on X in fp32, those of three nothing visible in bf16 and little where sums
// are long. Error over that of steps on X, 1 step | 3: 65 x 65 0.7 | 2.2, 160 x 1,900 0.7 | 1.5, 200 x 200 0.5 | 1.4,
// 256 x 256 0.5 | 1.3, 256 x 632 0.5 | 1.0, 512 x 512 0.5 | 1.1, 1,024 x 1,536 0.4 | 0.8; us, one of 64 x 64 76 | 92, 2,000
// of 100 x 100 1,425 | 1,584, 200 of 128 x 1,024 876 | 567, one of 256 x 632 127 | 123, 110 matrices of a model 19,200 |
// 14,600. Matrices of both kinds are taken in groups of their own, so that a matrix's result is a matter of itself alone.
enum Pick { kAll, kLongSides, kShortSides };
bool picked(Pick pick, int64_t rows, int64_t cols) {
  return rows * cols != 0 && (pick == kAll || (std::min(rows, cols) < kLongSide) == (pick == kShortSides));
}

// As many matrices as kGroupBytes hold, or fewer where their tiles fill the card better: 21 matrices of 1,024 x 2,438 (756
// tiles, two rounds of which the second is half empty) take 110 us a product, 14 of them 55. All that are left are taken at
// once unless two groups are better.
Group group_from(int64_t i, int64_t n, const int64_t* rows, const int64_t* cols, Pick pick) {
  Group g = {i, 0, 0, 0}, best = g;
  int64_t tiles = 0, best_tiles = 0;
  bool all = true;
  for (; g.end < n; ++g.end) {
    if (!picked(pick, rows[g.end], cols[g.end])) continue;
    const size_t bytes = planes_bytes(rows[g.end], cols[g.end]);
    if (g.count && g.planes + bytes > kGroupBytes) {
      all = false;
      break;
    }
    g.planes += bytes;
    g.sums += norm_blocks(rows[g.end], cols[g.end]);
    ++g.count;
    tiles += square_tiles(std::min(rows[g.end], cols[g.end]), kTile);
    if (best_tiles == 0 || tiles * cost(best_tiles) >= best_tiles * cost(tiles)) {
      best = g;
      ++best.end;
      best_tiles = tiles;
    }
  }
  return all && cost(tiles) <= cost(best_tiles) + cost(tiles - best_tiles) ? g : best;
}

// Bounds of what the steps form, from singular values in [0, 1], and the powers of two that bring them below 2^15.
struct Bounds {
  double x[kMaxSteps + 1], p[kMaxSteps];  // |X| before step k, |P| of step k
};

double poly(double a, double b, double c, double t) { return a + b * t + c * t * t; }

bool bounds_of(int steps, double a, double b, double c, Bounds* o) {
  if (steps < 1 || steps > kMaxSteps || !isfinite(a) || !isfinite(b) || !isfinite(c)) return false;
  o->x[0] = 1.0;
  for (int k = 0; k < steps; ++k) {
    const double s = o->x[k], top = s * s;
    double p = fmax(fabs(a), fabs(poly(a, b, c, top)));
    if (c != 0.0 && -b / (2 * c) > 0.0 && -b / (2 * c) < top) p = fmax(p, fabs(poly(a, b, c, -b / (2 * c))));
    double x = s * fabs(poly(a, b, c, top));
    const double d = 9 * b * b - 20 * a * c;  // a + 3 b t + 5 c t^2 = 0
    if (d >= 0.0) {
      const double w = sqrt(d);
      const double roots[3] = {c != 0.0 ? (-3 * b + w) / (10 * c) : -1.0, c != 0.0 ? (-3 * b - w) / (10 * c) : -1.0,
                               c == 0.0 && b != 0.0 ? -a / (3 * b) : -1.0};
      for (double t : roots)
        if (t > 0.0 && t < top) x = fmax(x, sqrt(t) * fabs(poly(a, b, c, t)));
    }
    if (!(p <= kMaxBound) || !(x <= kMaxBound)) return false;
    o->p[k] = p;
    o->x[k + 1] = x;
  }
  return true;
}

float scale_for(double bound) { return (float)exp2(14.0 - ceil(log2(fmax(bound, 1e-3)))); }

template <int TILE>
struct Launch {
  const Mat* mats;
  int count, squares, applies;  // matrices, tiles
  const Update& u;
  hipStream_t s;
  template <int KIND>
  void run(const Product& q, int jobs = 1) const {
    const int tiles = KIND <= kSquare ? squares : applies;
    const unsigned blocks = (unsigned)(cdiv(tiles, 8 * kRun) * 8 * kRun);
    fl_muon_product_kernel<KIND, TILE><<<dim3(blocks, (unsigned)jobs), threads_of<TILE>(), 0, s>>>(mats, count, tiles, q, u);
  }
};

// The steps of a group whose X is laid out, at most `stage` between two products with X.
template <int TILE>
void newton_schulz(const Launch<TILE>& launch, int stage, int steps, double a, double b, double c, const Bounds& bounds) {
  const int stages = (int)cdiv(steps, stage);
  float x_scale = scale_for(1.0);
  int source = 0;
  for (int st = 0, k = 0; st < stages; ++st) {
    const int len = (int)cdiv(steps - k, stages - st);  // the first ones are the longer ones
    // squares: 0 A, 1 U = A P, the others in turn P and the product of the P so far
    int poly_at = 2, product_at = -1, spare = 3;
    double product_bound = 0.0;
    float a_scale = scale_for(bounds.x[k] * bounds.x[k]), product_scale = 0.f;
    Product q = {};
    q.norm[0] = 1.f / (x_scale * x_scale);
    q.out_scale[0] = a_scale;
    launch.template run<kGram>(q);
    for (int e = 0; e < len; ++e, ++k) {
      const float p_scale = scale_for(bounds.p[k]);
      const bool last = e + 1 == len;
      q = {};
      q.out[0] = poly_at;
      q.norm[0] = 1.f / (a_scale * a_scale);
      q.a = (float)a;
      q.b = (float)b;
      q.c = (float)c;
      q.in_scale = 1.f / a_scale;
      q.out_scale[0] = p_scale;
      launch.template run<kPoly>(q);
      q = {};
      int jobs = 0;
      const float u_scale = scale_for(bounds.x[k] * bounds.x[k] * bounds.p[k]);
      const auto product = [&](int left, float left_scale, int out, float out_scale) {
        q.left[jobs] = left;
        q.right[jobs] = poly_at;
        q.out[jobs] = out;
        q.norm[jobs] = 1.f / (left_scale * p_scale);
        q.out_scale[jobs] = out_scale;
        ++jobs;
      };
      if (!last) product(0, a_scale, 1, u_scale);
      if (e == 0) {
        product_at = poly_at;
        product_scale = p_scale;
        product_bound = bounds.p[k];
      } else {
        product_bound *= bounds.p[k];
        const float scale = scale_for(product_bound);
        product(product_at, product_scale, spare, scale);
        const int old = product_at;
        product_at = spare;
        spare = old;
        product_scale = scale;
      }
      if (jobs) launch.template run<kSquare>(q, jobs);
      if (!last) {  // A = U P
        q = {};
        jobs = 0;
        a_scale = scale_for(bounds.x[k + 1] * bounds.x[k + 1]);
        product(1, u_scale, 0, a_scale);
        launch.template run<kSquare>(q);
        if (e == 0) poly_at = 4;
      }
    }
    q = {};
    q.left[0] = product_at;
    q.source = source;
    q.norm[0] = 1.f / (product_scale * x_scale);
    if (k < steps) {
      x_scale = scale_for(bounds.x[k]);
      q.out_scale[0] = x_scale;
      launch.template run<kApply>(q);
      source = 1 - source;
    } else {
      launch.template run<kFinal>(q);
    }
  }
}

int run(Pick pick, int64_t n, const void* const* g, void* const* p, float* const* buf, const int64_t* rows,
        const int64_t* cols, const double* lr_scale, int steps, double a, double b, double c, double eps, const Update& u, void* workspace,
        hipStream_t s) {
  Bounds bounds;
  if (!bounds_of(steps, a, b, c, &bounds)) return FL_ERR_INVALID_ARGUMENT;
  std::vector<int64_t> order;
  for (int64_t from = 0; from < n;) {
    const Group group = group_from(from, n, rows, cols, pick);
    if (group.count == 0) break;
    order.clear();
    for (int64_t i = from; i < group.end; ++i)
      if (picked(pick, rows[i], cols[i])) order.push_back(i);
    from = group.end;
    // the longest first, whose tiles take longest
    std::stable_sort(order.begin(), order.end(), [&](int64_t i, int64_t j) {
      return std::max(rows[i], cols[i]) > std::max(rows[j], cols[j]);
    });
    // small tiles while the large ones leave most of the card idle. us, 64 | 128: 36 tiles of 128 (1,024 x 1,024) 291 | 550,
    // 72 494 | 555, 108 569 | 565, 144 767 | 616, 200 (20 matrices of 400 x 400) 445 | 396
    int64_t large = 0;
    for (int64_t i : order) large += square_tiles(std::min(rows[i], cols[i]), kTile);
    const int tile = large >= 100 ? kTile : kSmallTile;
    char* at = static_cast<char*>(workspace);
    half_t* planes = reinterpret_cast<half_t*>(at);
    double* sums = reinterpret_cast<double*>(at + group.planes);
    Mat* mats = reinterpret_cast<Mat*>(at + group.planes + (size_t)group.sums * 8);
    int64_t first_norm = 0, first_copy = 0, first_square = 0, first_apply = 0, done = 0;
    Table t = {};
    for (int64_t i : order) {
      Mat& k = t.mat[t.n++];
      const bool tall = rows[i] > cols[i];
      k.base = planes;
      k.g = g[i];
      k.buf = buf ? buf[i] : nullptr;
      k.p = p[i];
      k.m = (int)(tall ? cols[i] : rows[i]);
      k.n = (int)(tall ? rows[i] : cols[i]);
      k.tall = tall;
      k.lr_scale = lr_scale ? (float)lr_scale[i] : 1.f;
      k.first_norm = (int)first_norm;
      k.first_copy = (int)first_copy;
      k.first_square = (int)first_square;
      k.first_apply = (int)first_apply;
      planes += planes_bytes(rows[i], cols[i]) / sizeof(half_t);
      first_norm += norm_blocks(rows[i], cols[i]);
      first_copy += cdiv(padded(rows[i]), kCopyTile) * cdiv(padded(cols[i]), kCopyTile);
      first_square += square_tiles(k.m, tile);
      first_apply += cdiv(k.m, tile) * cdiv(k.n, tile);
      if (t.n == kTable || done + t.n == group.count) {
        fl_muon_table_kernel<<<1, 64, 0, s>>>(t, mats + done);
        done += t.n;
        t.n = 0;
      }
    }
    const int count = (int)group.count;
    fl_muon_norm_kernel<<<(unsigned)first_norm, 256, 0, s>>>(mats, count, u, sums);
    fl_muon_copy_kernel<<<(unsigned)first_copy, 256, 0, s>>>(mats, count, u, sums, eps, scale_for(1.0));
    const int squares = (int)first_square, applies = (int)first_apply, stage = pick == kShortSides ? 1 : kStage;
    if (tile == kTile)
      newton_schulz(Launch<kTile>{mats, count, squares, applies, u, s}, stage, steps, a, b, c, bounds);
    else
      newton_schulz(Launch<kSmallTile>{mats, count, squares, applies, u, s}, stage, steps, a, b, c, bounds);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return hip_status(e);
  }
  return FL_OK;
}

int run(int64_t n, const void* const* g, void* const* p, float* const* buf, const int64_t* rows, const int64_t* cols,
        const double* lr_scale, int steps, double a, double b, double c, double eps, const Update& u, void* workspace,
        hipStream_t s) {
  const auto of = [&](Pick pick) {
    return run(pick, n, g, p, buf, rows, cols, lr_scale, steps, a, b, c, eps, u, workspace, s);
  };
  if (u.is_bf16) return of(kAll);
  const int status = of(kLongSides);
  return status == FL_OK ? of(kShortSides) : status;
}

// no exception leaves a C entry (the host's lists are all that allocates)
template <typename F>
int caught(F f) {
  try {
    return f();
  } catch (...) {
    return FL_ERR_HIP_BASE + (int)hipErrorOutOfMemory;
  }
}

bool addresses_ok(int64_t n, const void* const* p, const int64_t* rows, const int64_t* cols, size_t size) {
  if (!p) return false;
  for (int64_t i = 0; i < n; ++i)
    if (rows[i] * cols[i] > 0 && (!p[i] || !aligned(p[i], size))) return false;
  return true;
}

}  // namespace

extern "C" {

size_t fl_orthogonalize_workspace_bytes(int64_t n, const int64_t* rows, const int64_t* cols) {
  if (!lists_ok(n, rows, cols)) return 0;
  size_t most = 256;
  for (Pick pick : {kAll, kLongSides, kShortSides})
    for (int64_t i = 0; i < n;) {
      const Group g = group_from(i, n, rows, cols, pick);
      most = g.bytes() > most ? g.bytes() : most;
      i = g.end;
    }
  return most;
}

int fl_orthogonalize_check(int steps, double a, double b, double c) {
  Bounds bounds;
  return bounds_of(steps, a, b, c, &bounds) ? FL_OK : FL_ERR_INVALID_ARGUMENT;
}

int fl_orthogonalize(int64_t n, const void* const* x, int dtype, const int64_t* rows, const int64_t* cols, int steps,
                     double a, double b, double c, double eps, void* const* out, void* workspace,
                     size_t workspace_bytes, void* stream) {
  if (!dtype_ok(dtype)) return FL_ERR_DTYPE;
  if (!lists_ok(n, rows, cols) || !addresses_ok(n, x, rows, cols, esize(dtype)) ||
      !addresses_ok(n, (const void* const*)out, rows, cols, esize(dtype)) || !(eps >= 0.0))
    return FL_ERR_INVALID_ARGUMENT;
  if (!workspace || workspace_bytes < fl_orthogonalize_workspace_bytes(n, rows, cols)) return FL_ERR_WORKSPACE;
  if (!aligned(workspace, 16)) return FL_ERR_INVALID_ARGUMENT;
  Update u = {};
  u.is_bf16 = dtype == FL_DTYPE_BF16;
  return caught([&] {
    return run(n, x, out, nullptr, rows, cols, nullptr, steps, a, b, c, eps, u, workspace,
               static_cast<hipStream_t>(stream));
  });
}

int fl_muon_step(int64_t n, void* const* params, const void* const* grads, int dtype, float* const* buffers,
                 const int64_t* rows, const int64_t* cols, double lr, const float* lr_ptr, const double* lr_scale,
                 double momentum, int nesterov, double weight_decay, int steps, double a, double b, double c, double eps,
                 const float* grad_scale, void* workspace, size_t workspace_bytes, void* stream) {
  if (!dtype_ok(dtype)) return FL_ERR_DTYPE;
  if (!lists_ok(n, rows, cols) || !addresses_ok(n, (const void* const*)params, rows, cols, esize(dtype)) ||
      !addresses_ok(n, grads, rows, cols, esize(dtype)) ||
      !addresses_ok(n, (const void* const*)buffers, rows, cols, 4) || !(eps >= 0.0) || !lr_scale ||
      !(momentum >= 0.0 && momentum < 1.0) || !aligned(lr_ptr, 4) || !aligned(grad_scale, 4))
    return FL_ERR_INVALID_ARGUMENT;
  if (!workspace || workspace_bytes < fl_orthogonalize_workspace_bytes(n, rows, cols)) return FL_ERR_WORKSPACE;
  if (!aligned(workspace, 16)) return FL_ERR_INVALID_ARGUMENT;
  Update u = {};
  u.is_bf16 = dtype == FL_DTYPE_BF16;
  u.muon = 1;
  u.mu = (float)momentum;
  u.keep = (float)(1.0 - momentum);
  u.nesterov = nesterov != 0;
  u.grad_scale = grad_scale;
  u.lr_ptr = lr_ptr;
  u.lr = (float)lr;
  u.decay = (float)weight_decay;
  return caught([&] {
    return run(n, grads, params, buffers, rows, cols, lr_scale, steps, a, b, c, eps, u, workspace,
               static_cast<hipStream_t>(stream));
  });
}

}  // extern "C"
