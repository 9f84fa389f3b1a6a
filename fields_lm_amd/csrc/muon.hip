// muon.hip — matrices brought near their closest semi-orthogonal ones by Newton-Schulz steps, on their own and in a Muon
// step over many matrices at once.
//
//   X = G / (|G|_F + eps), then `steps` times X <- a X + (b A + c A^2) X with A = X X^T.
//
// A tall matrix is taken transposed, so that X is m x n with m <= n. The steps run on the m x m side: with
// P = a I + b A + c A^2 a step is X <- P X and makes A into P A P, and all of these commute and are symmetric. So k steps
// are one product X X^T, products of symmetric matrices (of which the lower half is computed) and one product
// (P_k .. P_1) X. A's small eigenvalues are squares of X's singular values, and a step lets their error grow a^2-fold
// (12 for the usual a) where X's own grows a-fold: after at most kStage steps X is formed and A taken from it anew,
// which keeps results as near to the formula's as steps on X in fp32 are.
//
// Every matrix is held as two fp16 planes, high and low part of its values times a power of two (22 bits), and a product
// is three of matrix instructions, high high + high low + low high, summed in fp32: bf16 operands end 3% from the result
// where singular values are alike, and as far as it is long where a few are strong.
#include "fl_common.h"

#include <math.h>

namespace {

using namespace fl;

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 half_t;

constexpr int kStage = 3;      // steps between two products with X
constexpr int kPad = 32;       // rows of planes are a multiple of this long, zeros behind the matrix
constexpr int kSquares = 5;    // m x m matrices of the workspace
constexpr int kTile = 128;     // rows and columns of a product's tile
constexpr int kCopyTile = 64;  // of the tile that is laid out by a block
constexpr int kTable = 56;     // matrices to a launch that sets up their table
constexpr int kNormChunk = 16384;  // values of a block of the norm
constexpr int64_t kMaxMatrices = 1 << 20, kMaxSide = 1 << 20, kMaxValues = (int64_t)1 << 30;
constexpr size_t kGroupBytes = (size_t)1 << 30;  // matrices are taken in groups of about this much workspace
constexpr int kMaxSteps = 64;
constexpr double kMaxBound = 1024.0;  // of singular values

struct Mat {
  half_t* base;    // its planes: X [m, ldn], X^T [n, ldm] twice, squares [m, ldm], each high then low
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

// the matrix whose blocks, counted by FIRST, hold `block`: as many begin at or before it, less one
template <int Mat::*FIRST>
__device__ __forceinline__ int matrix_of(const Mat* mats, int n, int block) {
  const int lane = threadIdx.x & 63;
  int begun = 0;
  for (int i = 0; i < n; i += 64) begun += __popcll(__ballot(i + lane < n && mats[min(i + lane, n - 1)].*FIRST <= block));
  return uniform(begun - 1);
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

// The momentum's update (Muon) and the sum of the squares of what is orthogonalized, in fp64.
__global__ __launch_bounds__(256) void fl_muon_norm_kernel(const Mat* __restrict__ mats, int n, const Update u,
                                                           double* __restrict__ part) {
  __shared__ double s_sum[4];
  const int i = matrix_of<&Mat::first_norm>(mats, n, blockIdx.x);
  const Mat& k = mats[i];
  const int64_t numel = (int64_t)k.m * k.n, lo = (int64_t)((int)blockIdx.x - k.first_norm) * kNormChunk;
  const int64_t hi = lo + kNormChunk < numel ? lo + kNormChunk : numel;
  const float scale = u.grad_scale ? *u.grad_scale : 1.f;
  const bool skip = skipped(u);
  double sum = 0.0;
  for (int64_t j = lo + threadIdx.x; j < hi; j += 256) {
    float v = load_any(k.g, j, u.is_bf16);
    if (u.muon) {
      v *= scale;
      const float b = fmaf(u.mu, k.buf[j], u.keep * v);
      if (!skip) k.buf[j] = b;
      v = u.nesterov ? fmaf(u.keep, v, u.mu * b) : b;
    }
    sum = fma((double)v, (double)v, sum);
  }
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) sum += __shfl_xor(sum, d);
  if ((threadIdx.x & 63) == 0) s_sum[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) part[blockIdx.x] = (s_sum[0] + s_sum[1]) + (s_sum[2] + s_sum[3]);
}

// high and low part of v
__device__ __forceinline__ void split(float v, half_t& hi, half_t& lo) {
  hi = (half_t)v;
  lo = (half_t)(v - (float)hi);
}

// X = G / (|G| + eps) times x_scale, as planes of X and of X^T, a tile of 64 x 64 to a block.
__global__ __launch_bounds__(256) void fl_muon_copy_kernel(const Mat* __restrict__ mats, int n, const Update u,
                                                           const double* __restrict__ part, double eps, float x_scale) {
  __shared__ float s_x[kCopyTile][kCopyTile + 1];
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
  const double inv = (double)x_scale / (sqrt(sum) + eps);

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
  const int64_t plane_s = rows * ld_r, plane_t = cols * ld_c;
  for (int j = threadIdx.x; j < kCopyTile * kCopyTile; j += 256) {
    const int r = r0 + j / kCopyTile, c = c0 + j % kCopyTile;
    float v = 0.f;
    if (r < rows && c < cols) {
      const int64_t at = (int64_t)r * cols + c;
      v = load_any(k.g, at, u.is_bf16);
      if (u.muon) {
        const float b = k.buf[at];
        v = u.nesterov ? fmaf(u.keep, v * scale, u.mu * b) : b;
      }
      v = (float)((double)v * inv);
    }
    s_x[j / kCopyTile][j % kCopyTile] = v;
    if (r < rows && c < ld_r) {
      half_t hi, lo;
      split(v, hi, lo);
      straight[r * ld_r + c] = hi;
      straight[plane_s + r * ld_r + c] = lo;
    }
  }
  __syncthreads();
  for (int j = threadIdx.x; j < kCopyTile * kCopyTile; j += 256) {
    const int c = c0 + j / kCopyTile, r = r0 + j % kCopyTile;
    if (c < cols && r < ld_c) {
      half_t hi, lo;
      split(s_x[j % kCopyTile][j / kCopyTile], hi, lo);
      turned[c * ld_c + r] = hi;
      turned[plane_t + c * ld_c + r] = lo;
    }
  }
}

// What a product is formed of: L R^T of rows of X, of X^T or of a square.
struct Product {
  int left[2], right[2], out[2];  // squares' numbers, for up to two products of a launch
  int source;                     // which X^T
  float norm;                     // 1 / (the operands' scales)
  float a, b, c;                  // of the polynomial
  float in_scale, out_scale;      // of the square that it reads, and of the result
};

enum Kind { kGram, kPoly, kSquare, kApply, kFinal };

// One tile of L R^T. Rows past an operand's last are read as its last one; what they give is not written.
// The LDS holds two steps of 32 columns: while a step is multiplied the next one's rows are loaded straight into it. A
// row's four packs of 16 bytes change places by its number, so that eight rows' equal packs lie in different banks.
template <int KIND>
__global__ __launch_bounds__(256) void fl_muon_product_kernel(const Mat* __restrict__ mats, int n, const Product q,
                                                              const Update u) {
  constexpr bool kSymmetric = KIND <= kSquare;
  constexpr int kStep = 32, kRow = kStep * 2;  // halves, bytes
  constexpr int kPlane = kTile * kRow, kOperand = 2 * kPlane, kBuffer = 2 * kOperand;
  __shared__ __attribute__((aligned(16))) char s_tile[2 * kBuffer];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int job = blockIdx.y;
  const int which = kSymmetric ? matrix_of<&Mat::first_square>(mats, n, blockIdx.x)
                               : matrix_of<&Mat::first_apply>(mats, n, blockIdx.x);
  const Mat& k = mats[which];
  const int m = k.m, cols = k.n;
  const int64_t ldn = padded(cols), ldm = padded(m);
  half_t* x = k.base;
  half_t* xt[2] = {x + 2 * (int64_t)m * ldn, x + 2 * (int64_t)m * ldn + 2 * cols * ldm};
  half_t* squares = xt[1] + 2 * cols * ldm;
  const int64_t square = 2 * (int64_t)m * ldm;

  // operands: rows, their count, their length
  const half_t *lp, *rp;
  int l_rows, r_rows;
  int64_t ld;
  int ti, tj;
  const bool turn = KIND == kFinal && k.tall;
  if constexpr (kSymmetric) {
    const int t = (int)blockIdx.x - k.first_square;
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
    const int across = (r_rows + kTile - 1) / kTile, t = (int)blockIdx.x - k.first_apply;
    ti = t / across;
    tj = t - ti * across;
  }
  const int r0 = ti * kTile, c0 = tj * kTile;

  // 16 rows of one plane to an instruction: 16 instructions an operand and buffer, four to a wave and operand
  const int load_row = lane >> 2, load_pack = (lane & 3) ^ ((load_row >> 1) & 3);
  auto load = [&](int buffer, int step) {
#pragma unroll
    for (int o = 0; o < 2; ++o) {
      const half_t* base = o ? rp : lp;
      const int rows = o ? r_rows : l_rows, first = o ? c0 : r0;
      const int64_t plane = (int64_t)rows * ld;
#pragma unroll
      for (int j = 0; j < kTile / 32; ++j) {
        const int piece = wave * (kTile / 32) + j;  // of 2 planes x kTile / 16
        const int p = piece / (kTile / 16), rr = piece % (kTile / 16) * 16;
        const int row = min(first + rr + load_row, rows - 1);
        const half_t* from = base + p * plane + row * ld + step * kStep + load_pack * 8;
        __builtin_amdgcn_global_load_lds(
            (const __attribute__((address_space(1))) void*)from,
            (__attribute__((address_space(3))) void*)(s_tile + buffer * kBuffer + o * kOperand + p * kPlane + rr * kRow),
            16, 0, 0);
      }
    }
  };

  const int wr = (wave >> 1) * 64, wc = (wave & 1) * 64;
  f32x16 acc[2][2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;

  const int steps = (int)(ld / kStep);
  load(0, 0);
  for (int s = 0; s < steps; ++s) {
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();  // the step's rows are there, and nobody reads the other buffer any more
    if (s + 1 < steps) load((s + 1) & 1, s + 1);
    const char* buf = s_tile + (s & 1) * kBuffer;
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      f16x8 l[2][2], r[2][2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int lr = wr + i * 32 + (lane & 31), rr = wc + i * 32 + (lane & 31);
        const int pack = kk * 2 + (lane >> 5);
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          l[i][p] = *reinterpret_cast<const f16x8*>(buf + p * kPlane + lr * kRow + (pack ^ ((lr >> 1) & 3)) * 16);
          r[i][p] = *reinterpret_cast<const f16x8*>(buf + kOperand + p * kPlane + rr * kRow + (pack ^ ((rr >> 1) & 3)) * 16);
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(l[i][0], r[j][0], acc[i][j], 0, 0, 0);
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(l[i][0], r[j][1], acc[i][j], 0, 0, 0);
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(l[i][1], r[j][0], acc[i][j], 0, 0, 0);
        }
    }
  }

  const float lr = KIND == kFinal && u.muon ? (u.lr_ptr ? *u.lr_ptr : u.lr) : 0.f;
  const float keep = 1.f - lr * u.decay, rate = lr * k.lr_scale;
  const bool skip = KIND == kFinal && u.muon && skipped(u);
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int row = r0 + wr + i * 32 + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3);
        const int col = c0 + wc + j * 32 + (lane & 31);
        float v = acc[i][j][e] * q.norm;
        if constexpr (kSymmetric) {
          // the lower half and its mirror, with the zeros behind each row
          if (row < col || row >= ldm || col >= m) continue;
          const bool in = row < m;
          if constexpr (KIND == kPoly) {
            const half_t* from = squares + q.left[job] * square + (int64_t)(in ? row : 0) * ldm + col;
            v = q.b * ((float)from[0] + (float)from[m * ldm]) * q.in_scale + q.c * v + (row == col ? q.a : 0.f);
          }
          half_t hi, lo;
          split(in ? v * q.out_scale : 0.f, hi, lo);
          half_t* to = squares + q.out[job] * square;
          if (in) {
            to[row * ldm + col] = hi;
            to[(m + row) * ldm + col] = lo;
          }
          to[col * ldm + row] = hi;
          to[(m + col) * ldm + row] = lo;
        } else if constexpr (KIND == kApply) {
          // X and the other X^T
          const bool in = row < m && col < cols;
          half_t hi, lo;
          split(in ? v * q.out_scale : 0.f, hi, lo);
          if (row < m && col < ldn) {
            x[row * ldn + col] = hi;
            x[(m + row) * ldn + col] = lo;
          }
          half_t* to = xt[1 - q.source];
          if (col < cols && row < ldm) {
            to[col * ldm + row] = hi;
            to[((int64_t)cols + col) * ldm + row] = lo;
          }
        } else {
          if (row >= l_rows || col >= r_rows || skip) continue;
          const int64_t at = (int64_t)row * r_rows + col;
          if (u.muon) v = fmaf(-rate, v, load_any(k.p, at, u.is_bf16) * keep);
          if (u.is_bf16)
            store_as(static_cast<bf16_bits*>(k.p) + at, v);
          else
            store_as(static_cast<float*>(k.p) + at, v);
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

Group group_from(int64_t i, int64_t n, const int64_t* rows, const int64_t* cols) {
  Group g = {i, 0, 0, 0};
  for (; g.end < n; ++g.end) {
    if (rows[g.end] * cols[g.end] == 0) continue;
    const size_t bytes = planes_bytes(rows[g.end], cols[g.end]);
    if (g.count && g.planes + bytes > kGroupBytes) break;
    g.planes += bytes;
    g.sums += norm_blocks(rows[g.end], cols[g.end]);
    ++g.count;
  }
  return g;
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

int run(int64_t n, const void* const* g, void* const* p, float* const* buf, const int64_t* rows, const int64_t* cols,
        const double* lr_scale, int steps, double a, double b, double c, double eps, const Update& u, void* workspace,
        hipStream_t s) {
  Bounds bounds;
  if (!bounds_of(steps, a, b, c, &bounds)) return FL_ERR_INVALID_ARGUMENT;
  for (int64_t i = 0; i < n;) {
    const Group group = group_from(i, n, rows, cols);
    if (group.count == 0) break;
    char* at = static_cast<char*>(workspace);
    half_t* planes = reinterpret_cast<half_t*>(at);
    double* sums = reinterpret_cast<double*>(at + group.planes);
    Mat* mats = reinterpret_cast<Mat*>(at + group.planes + (size_t)group.sums * 8);
    int64_t first_norm = 0, first_copy = 0, first_square = 0, first_apply = 0, done = 0;
    Table t = {};
    for (; i < group.end; ++i) {
      if (rows[i] * cols[i] == 0) continue;
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
      const int64_t side = cdiv(k.m, kTile);
      first_square += side * (side + 1) / 2;
      first_apply += side * cdiv(k.n, kTile);
      if (t.n == kTable || i + 1 == group.end) {
        fl_muon_table_kernel<<<1, 64, 0, s>>>(t, mats + done);
        done += t.n;
        t.n = 0;
      }
    }
    if (t.n) {
      fl_muon_table_kernel<<<1, 64, 0, s>>>(t, mats + done);
      done += t.n;
    }
    const int count = (int)group.count;
    fl_muon_norm_kernel<<<(unsigned)first_norm, 256, 0, s>>>(mats, count, u, sums);
    float x_scale = scale_for(1.0);
    fl_muon_copy_kernel<<<(unsigned)first_copy, 256, 0, s>>>(mats, count, u, sums, eps, x_scale);
    int source = 0;
    const dim3 squares((unsigned)first_square), apply((unsigned)first_apply);
    const int stages = (int)cdiv(steps, kStage);
    for (int st = 0, k = 0; st < stages; ++st) {
      const int len = (steps - k + stages - st - 1) / (stages - st);  // the first ones are the longer ones
      // squares: A, U, then three in turn for P and the product of the P so far
      int poly_at = 2, product_at = -1, spare = 3, other = 4;
      double product_bound = 0.0;
      float a_scale = scale_for(bounds.x[k] * bounds.x[k]), product_scale = 0.f;
      Product q = {};
      q.out[0] = 0;
      q.norm = 1.f / (x_scale * x_scale);
      q.out_scale = a_scale;
      fl_muon_product_kernel<kGram><<<squares, 256, 0, s>>>(mats, count, q, u);
      for (int e = 0; e < len; ++e, ++k) {
        const float p_scale = scale_for(bounds.p[k]);
        q = {};
        q.left[0] = q.right[0] = 0;
        q.out[0] = poly_at;
        q.norm = 1.f / (a_scale * a_scale);
        q.a = (float)a;
        q.b = (float)b;
        q.c = (float)c;
        q.in_scale = 1.f / a_scale;
        q.out_scale = p_scale;
        fl_muon_product_kernel<kPoly><<<squares, 256, 0, s>>>(mats, count, q, u);
        const bool last = e + 1 == len;
        const float u_scale = scale_for(bounds.x[k] * bounds.x[k] * bounds.p[k]);
        if (!last) {  // U = A P
          q = {};
          q.left[0] = 0;
          q.right[0] = poly_at;
          q.out[0] = 1;
          q.norm = 1.f / (a_scale * p_scale);
          q.out_scale = u_scale;
          fl_muon_product_kernel<kSquare><<<squares, 256, 0, s>>>(mats, count, q, u);
        }
        if (product_at < 0) {
          product_at = poly_at;
          product_scale = p_scale;
          product_bound = bounds.p[k];
        } else {  // the product of the P
          product_bound *= bounds.p[k];
          const float scale = scale_for(product_bound);
          q = {};
          q.left[0] = product_at;
          q.right[0] = poly_at;
          q.out[0] = spare;
          q.norm = 1.f / (product_scale * p_scale);
          q.out_scale = scale;
          fl_muon_product_kernel<kSquare><<<squares, 256, 0, s>>>(mats, count, q, u);
          const int free_at = product_at;
          product_at = spare;
          spare = free_at;
          product_scale = scale;
        }
        if (!last) {  // A = U P
          const float next = scale_for(bounds.x[k + 1] * bounds.x[k + 1]);
          q = {};
          q.left[0] = 1;
          q.right[0] = poly_at;
          q.out[0] = 0;
          q.norm = 1.f / (u_scale * p_scale);
          q.out_scale = next;
          fl_muon_product_kernel<kSquare><<<squares, 256, 0, s>>>(mats, count, q, u);
          a_scale = next;
          if (product_at == poly_at) {
            poly_at = other;
          }
        }
      }
      q = {};
      q.left[0] = product_at;
      q.source = source;
      q.norm = 1.f / (product_scale * x_scale);
      if (k < steps) {
        x_scale = scale_for(bounds.x[k]);
        q.out_scale = x_scale;
        fl_muon_product_kernel<kApply><<<apply, 256, 0, s>>>(mats, count, q, u);
        source = 1 - source;
      } else {
        fl_muon_product_kernel<kFinal><<<apply, 256, 0, s>>>(mats, count, q, u);
      }
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return hip_status(e);
  }
  return FL_OK;
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
  for (int64_t i = 0; i < n;) {
    const Group g = group_from(i, n, rows, cols);
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
  return run(n, x, out, nullptr, rows, cols, nullptr, steps, a, b, c, eps, u, workspace,
             static_cast<hipStream_t>(stream));
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
  return run(n, grads, params, buffers, rows, cols, lr_scale, steps, a, b, c, eps, u, workspace,
             static_cast<hipStream_t>(stream));
}

}  // extern "C"
