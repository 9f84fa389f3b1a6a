// embedding.hip — rows of an embedding by token, scaled, and the gradient of its weight: with a scale s and the
// tokens k_n,
//   out[n] = s W[k_n],    dW[v] = s sum over n with k_n = v of g[n], in an order of the tokens' alone.
//
// Both directions are bound by memory, each row touched once: 8,192 tokens of 1,024 fp32 values take 12 us forward
// (5.4 TB/s), and with 16,384 rows 35 us back (100 MB: 18 us of sums at 5.7 TB/s behind 11 us of sorting, 6 us of joining
// shared rows); 32,768 tokens and 131,072 rows in bf16 23 us (5.8 TB/s) and 107 us (335 MB: 81 us of sums at 4.1 TB/s, 14 and
// 12). A row that many tokens share is joined by one wave: 32,768 tokens, 16,384 rows of 1,024 fp32 values, both directions,
// 97 us; with a quarter of the tokens alike 137, half of them 175, all 265 (as padding 80).
#include "fl_common.h"

#include <algorithm>

namespace {

using namespace fl;

constexpr int kMaxBuckets = 2048;
constexpr int kMaxRows = 4096;    // of a bucket
constexpr int kSortThreads = 512;
constexpr int kMaxChunks = 64;    // of the tokens, a block to each
constexpr int kOneChunk = 1024;  // tokens up to which one block sorts, without a launch that counts (2,048: 29.1 us a gradient
                                 // of 16,384 rows by itself, 26.6 in four blocks and two launches; 999 the same)
constexpr int kSumThreads = 256;
constexpr int kJoinThreads = 512;
constexpr int kPiece = 32;        // entries of a list that a block takes
constexpr int kAhead = 8;         // rows that a wave loads before it adds them
constexpr size_t kPartBytes = (size_t)1 << 28;  // of parts, about; pieces grow where they would take more
constexpr int64_t kMaxExtras = (int64_t)1 << 22;  // pieces behind their buckets' first: a launch's threads have to be fewer
                                                  // than 2^32, and the join takes kJoinThreads to each
constexpr int64_t kMaxTokens = (int64_t)1 << 30, kMaxVocab = (int64_t)kMaxBuckets * kMaxRows, kMaxDim = (int64_t)1 << 24;

// Streaming stores: a fifth less time for the gradient of 32,768 tokens, 131,072 rows of 1,024 in bf16; a third of that as
// fast either way.
__device__ __forceinline__ void store_once(u32x4_any* p, u32x4 v) { __builtin_nontemporal_store(v, p); }
__device__ __forceinline__ void store_once(u32x2_any* p, u32x2 v) { __builtin_nontemporal_store(v, p); }

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
      store_once(reinterpret_cast<u32x4_any*>(p), a);
      store_once(reinterpret_cast<u32x4_any*>(p + 4), b);
    } else {
      u32x4 a;
#pragma unroll
      for (int i = 0; i < 4; ++i) a[i] = bf16_pair(v[2 * i], v[2 * i + 1]);
      store_once(reinterpret_cast<u32x4_any*>(p), a);
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

// ---------------------------------------------------------------- the gradient
// (Every row's wave looking through all tokens instead, the simplest form: 708 us where this takes 57, forward included.)
// The vocabulary is cut into buckets of `1 << shift` rows, the tokens' places are put in order of their buckets, within one
// in their own order, and a block sums each bucket's rows: tokens, gradients and result are touched once. A list longer
// than a piece is shared by several blocks, whose sums another launch adds in the pieces' order, so that the grouping of
// sums is a matter of the tokens alone.

struct Entry {
  uint32_t at;   // the token's place
  uint32_t row;  // within the bucket
};

struct Sort {
  const int64_t* tokens;
  int64_t n, V, padding;
  int shift, buckets, chunk, chunks, piece;
  uint32_t* counts;    // [chunks, kMaxBuckets]
  uint32_t* starts;    // [buckets + 1]
  uint32_t* extra;     // [0] the number of pieces behind their buckets' first, then each one's bucket
  uint32_t* first;     // [buckets] a bucket's first extra piece
  uint32_t* present;   // [2 extras, rows / 32 rounded up] the rows that a piece has
  Entry* list;         // [n]
};

// the token's bucket, or -1 where it passes no gradient
__device__ __forceinline__ int bucket_of(const Sort& s, int64_t i, uint32_t& row) {
  const int64_t t = s.tokens[i];
  if (t < 0 || t >= s.V || t == s.padding) return -1;
  row = (uint32_t)t & ((1u << s.shift) - 1);
  return (int)(t >> s.shift);
}

__device__ __forceinline__ void count_tokens(const Sort& s, int chunk, uint32_t* s_count) {
  for (int b = threadIdx.x; b < kMaxBuckets; b += kSortThreads) s_count[b] = 0;
  __syncthreads();
  const int64_t lo = (int64_t)chunk * s.chunk, hi = lo + s.chunk < s.n ? lo + s.chunk : s.n;
  for (int64_t i = lo + threadIdx.x; i < hi; i += kSortThreads) {
    uint32_t row;
    const int b = bucket_of(s, i, row);
    if (b >= 0) atomicAdd(&s_count[b], 1u);
  }
  __syncthreads();
}

__global__ __launch_bounds__(kSortThreads) void fl_embedding_count_kernel(const Sort s) {
  __shared__ uint32_t s_count[kMaxBuckets];
  count_tokens(s, (int)blockIdx.x, s_count);
  for (int b = threadIdx.x; b < kMaxBuckets; b += kSortThreads) s.counts[blockIdx.x * kMaxBuckets + b] = s_count[b];
}

// exclusive sums over the block's threads
__device__ uint32_t block_scan(uint32_t v, uint32_t* s_wave) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t sum = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t o = __shfl_up(sum, d);
    if (lane >= d) sum += o;
  }
  __syncthreads();
  if (lane == 63) s_wave[wave] = sum;
  __syncthreads();
  uint32_t before = 0;
  for (int i = 0; i < wave; ++i) before += s_wave[i];
  return before + sum - v;
}

// A chunk's tokens to their buckets' lists. Where each begins is summed from all chunks' counts by every block for itself
// (a launch less). A round of 512 tokens takes its places wave by wave, so that they come in order.
__global__ __launch_bounds__(kSortThreads) void fl_embedding_sort_kernel(const Sort s) {
  __shared__ uint32_t s_next[kMaxBuckets], s_wave[kSortThreads / 64];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  constexpr int kPer = kMaxBuckets / kSortThreads;
  if (s.chunks == 1) count_tokens(s, 0, s_next);
  uint32_t total[kPer], before[kPer];
  const int b0 = threadIdx.x * kPer;  // consecutive buckets to a thread
  const int64_t lo = (int64_t)blockIdx.x * s.chunk, hi = lo + s.chunk < s.n ? lo + s.chunk : s.n;
  uint32_t row = 0, next_row = 0;
  int b = lo + threadIdx.x < hi ? bucket_of(s, lo + threadIdx.x, row) : -1, next = -1;
  if (s.chunks == 1) {
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      total[k] = s_next[b0 + k];
      before[k] = 0;
    }
  } else {
    static_assert(kPer == 4, "");
    u32x4 all = {0, 0, 0, 0}, mine = {0, 0, 0, 0};
    const u32x4* counts = reinterpret_cast<const u32x4*>(s.counts) + threadIdx.x;
#pragma unroll 8
    for (int c = 0; c < s.chunks; ++c) {
      const u32x4 v = counts[c * (kMaxBuckets / 4)];
      if (c == (int)blockIdx.x) mine = all;
      all += v;
    }
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      total[k] = all[k];
      before[k] = mine[k];
    }
  }
  uint32_t mine = 0;
#pragma unroll
  for (int k = 0; k < kPer; ++k) mine += total[k];
  uint32_t start = block_scan(mine, s_wave);  // (its barriers stand between the counts' last reads and s_next's writes)
  if (blockIdx.x == 0) {
    uint32_t more = 0;
#pragma unroll
    for (int k = 0; k < kPer; ++k) more += total[k] > (uint32_t)s.piece ? (total[k] - 1) / (uint32_t)s.piece : 0;
    uint32_t at = block_scan(more, s_wave), begin = start;
    if (threadIdx.x == kSortThreads - 1) {
      s.extra[0] = at + more;
      s.starts[s.buckets] = start + mine;
    }
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      if (b0 + k >= s.buckets) continue;
      s.starts[b0 + k] = begin;
      s.first[b0 + k] = at;
      const uint32_t pieces = total[k] > (uint32_t)s.piece ? (total[k] - 1) / (uint32_t)s.piece : 0;
      for (uint32_t j = 0; j < pieces; ++j) s.extra[1 + at + j] = (uint32_t)(b0 + k);
      at += pieces;
      begin += total[k];
    }
  }
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    if (b0 + k < s.buckets) s_next[b0 + k] = start + before[k];
    start += total[k];
  }
  __syncthreads();
  for (int64_t at = lo; at < hi; at += kSortThreads) {
    const int64_t i = at + threadIdx.x;
    next = i + kSortThreads < hi ? bucket_of(s, i + kSortThreads, next_row) : -1;
    // the lanes of the same bucket
    uint64_t same = __ballot(b >= 0);
    for (int bit = 0; 1 << bit < s.buckets; ++bit) {
      const uint64_t set = __ballot(b >= 0 && (b >> bit & 1));
      same &= b >> bit & 1 ? set : ~set;
    }
    const int rank = __popcll(same & ((1ull << lane) - 1));
    uint32_t to = 0;
    for (int w = 0; w < kSortThreads / 64; ++w) {
      if (w == wave && b >= 0) {
        to = s_next[b] + rank;
        if (rank == 0) s_next[b] = to + __popcll(same);
      }
      __syncthreads();
    }
    if (b >= 0) s.list[to] = Entry{(uint32_t)i, row};
    b = next;
    row = next_row;
  }
}

// N values of a row as they lie, `left` of them there, 8 bytes or a multiple of 16
template <int N, typename T>
struct Pack {
  static constexpr int kWords = N * (int)sizeof(T) / 4;
  uint32_t w[kWords];
  __device__ __forceinline__ void load(const T* p, int64_t left) {
    if (left >= N) {
      if constexpr (kWords >= 4) {
#pragma unroll
        for (int q = 0; q < kWords; q += 4) {
          const u32x4 r = *reinterpret_cast<const u32x4_any*>(p + q * 4 / (int)sizeof(T));
#pragma unroll
          for (int i = 0; i < 4; ++i) w[q + i] = r[i];
        }
      } else {
        const u32x2 r = *reinterpret_cast<const u32x2_any*>(p);
        w[0] = r[0];
        w[1] = r[1];
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = 0;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < left) {
        if constexpr (sizeof(T) == 4)
          w[i] = __float_as_uint(p[i]);
        else
          w[i >> 1] |= (uint32_t)p[i] << (16 * (i & 1));
      }
  }
  __device__ __forceinline__ float operator[](int i) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
    return i & 1 ? bf16_hi(w[i >> 1]) : bf16_lo(w[i >> 1]);
  }
};
template <int N, typename T>
__device__ __forceinline__ void store_values(T* p, int64_t left, const float* v) {
  if (left >= N) {
    if constexpr (N == 8) {
      store8(p, left, v);
    } else if constexpr (sizeof(T) == 4) {
      store_once(reinterpret_cast<u32x4_any*>(p),
                 u32x4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])});
    } else {
      store_once(reinterpret_cast<u32x2_any*>(p), u32x2{bf16_pair(v[0], v[1]), bf16_pair(v[2], v[3])});
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < left) store_as(p + i, v[i]);
  }
}

// acc plus the rows `base + at(bit) * D` of the bits of `mine`, lowest first, kAhead of them loaded before they are added
template <typename T, int N, typename At>
__device__ __forceinline__ void add_rows(uint64_t mine, const T* base, int64_t D, int64_t left, At at, float* acc) {
  while (mine) {
    Pack<N, T> v[kAhead];
    int got = 0;
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (mine) {
        const int l = __ffsll((unsigned long long)mine) - 1;
        mine &= mine - 1;
        v[u].load(base + at(l) * D, left);
        got = u + 1;
      }
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (u < got) {
#pragma unroll
        for (int i = 0; i < N; ++i) acc[i] += v[u][i];
      }
  }
}

// The sums of a piece of a bucket's list, a wave to a row and 64 N columns in turn, N values being 16 bytes of the wider of
// both types. The extra pieces' blocks come first, since they take longest. Where the bucket
// has one piece they are the result, rows of no entry among them as zeros. Else they go to `part`, a place to every piece
// and row, and which rows it has to `present`.
template <typename GT, typename WT>
__global__ __launch_bounds__(kSumThreads) void fl_embedding_sum_kernel(const Sort s, int extras,
                                                                       const GT* __restrict__ g, int64_t D, float scale,
                                                                       float* __restrict__ part,
                                                                       WT* __restrict__ out) {
  constexpr int N = sizeof(GT) == 2 && sizeof(WT) == 2 ? 8 : 4, kColumns = 64 * N;
  __shared__ uint32_t s_present[kMaxRows / 32];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  int bucket = (int)blockIdx.x - extras;
  uint32_t piece = 0;
  if (bucket < 0) {
    const uint32_t j = blockIdx.x;
    if (j >= s.extra[0]) return;
    bucket = (int)s.extra[1 + j];
    piece = j - s.first[bucket] + 1;
  }
  bucket = uniform(bucket);
  piece = uniform((int)piece);
  const uint32_t begin = s.starts[bucket], end = s.starts[bucket + 1];
  const uint32_t pieces = end - begin > (uint32_t)s.piece ? (end - begin - 1) / (uint32_t)s.piece + 1 : 1;
  const uint32_t lo = begin + piece * (uint32_t)s.piece, hi = min(lo + (uint32_t)s.piece, end);
  const int64_t row0 = (int64_t)bucket << s.shift;
  const int rows = (int)min((int64_t)1 << s.shift, s.V - row0), words = (rows + 31) / 32;
  const int slices = (int)((D + kColumns - 1) / kColumns);
  const bool alone = pieces == 1;
  // a shared bucket's places: it has at most two pieces to an extra one
  const int64_t place = (int64_t)s.first[bucket] * 2;
  float* parts = part + (place << s.shift) * D;
  uint32_t* present = s.present + place * ((((int64_t)1 << s.shift) + 31) / 32);
  Entry e = {0, 0xffffffffu};
  if (lo + lane < hi) e = s.list[lo + lane];
  if (!alone) {
    for (int w = threadIdx.x; w < words; w += kSumThreads) s_present[w] = 0;
    __syncthreads();
    for (uint32_t at = lo + threadIdx.x; at < hi; at += kSumThreads) {
      const uint32_t row = s.list[at].row;
      atomicOr(&s_present[row >> 5], 1u << (row & 31));
    }
    __syncthreads();
    for (int w = threadIdx.x; w < words; w += kSumThreads) present[(int64_t)piece * words + w] = s_present[w];
  }
  for (int unit = wave; unit < rows * slices; unit += kSumThreads / 64) {
    const int row = unit / slices, slice = unit - row * slices;
    if (!alone && !(s_present[row >> 5] >> (row & 31) & 1)) continue;
    const int64_t c = (int64_t)slice * kColumns + lane * N;
    float acc[N] = {};
    for (uint32_t at = lo; at < hi; at += 64) {
      Entry x = e;
      if (hi - lo > 64) {
        x = Entry{0, 0xffffffffu};
        if (at + lane < hi) x = s.list[at + lane];
      }
      const uint64_t mine = __ballot(x.row == (uint32_t)row);
      if (c < D)
        add_rows<GT, N>(mine, g + c, D, D - c,
                        [&](int l) { return (int64_t)(uint32_t)__builtin_amdgcn_readlane((int)x.at, l); }, acc);
    }
    if (c < D) {
      if (alone) {
#pragma unroll
        for (int k = 0; k < N; ++k) acc[k] *= scale;
        store_values<N>(out + (row0 + row) * D + c, D - c, acc);
      } else {
        store_values<N>(parts + ((int64_t)piece * rows + row) * D + c, D - c, acc);
      }
    }
  }
}

// The rows of the buckets that several blocks shared: a block to a quarter of a bucket's rows adds the pieces that have
// them, in their order. (Left to the last of those blocks instead, each had to write its cache back before it could say
// that it was done: 8,192 tokens of 1,024 fp32 values took 49 us in all, 32 with pieces twice as long, 24 so.)
template <int N, typename WT>
__global__ __launch_bounds__(kJoinThreads) void fl_embedding_join_kernel(const Sort s, int64_t D, float scale,
                                                                         const float* __restrict__ part,
                                                                         WT* __restrict__ out) {
  constexpr int kColumns = 64 * N;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  if (blockIdx.x >= s.extra[0]) return;
  const int bucket = uniform((int)s.extra[1 + blockIdx.x]);
  if (s.first[bucket] != blockIdx.x) return;
  const uint32_t count = s.starts[bucket + 1] - s.starts[bucket];
  const uint32_t pieces = (count - 1) / (uint32_t)s.piece + 1;
  const int64_t row0 = (int64_t)bucket << s.shift;
  const int rows = (int)min((int64_t)1 << s.shift, s.V - row0), words = (rows + 31) / 32;
  const int slices = (int)((D + kColumns - 1) / kColumns);
  const int64_t place = (int64_t)blockIdx.x * 2;
  const float* parts = part + (place << s.shift) * D;
  const uint32_t* present = s.present + place * ((((int64_t)1 << s.shift) + 31) / 32);
  constexpr int kWaves = kJoinThreads / 64;
  for (int unit = (int)blockIdx.y * kWaves + wave; unit < rows * slices; unit += (int)gridDim.y * kWaves) {
    const int row = unit / slices, slice = unit - row * slices;
    const int64_t c = (int64_t)slice * kColumns + lane * N;
    float acc[N] = {};
    for (uint32_t j = 0; j < pieces; j += 64) {
      const bool has = j + lane < pieces && (present[(int64_t)(j + lane) * words + (row >> 5)] >> (row & 31) & 1);
      const uint64_t mine = __ballot(has);
      if (c < D)
        add_rows<float, N>(mine, parts + ((int64_t)j * rows + row) * D + c, D, D - c,
                           [&](int l) { return (int64_t)l * rows; }, acc);
    }
    if (c < D) {
#pragma unroll
      for (int k = 0; k < N; ++k) acc[k] *= scale;
      store_values<N>(out + (row0 + row) * D + c, D - c, acc);
    }
  }
}

template <typename WT, typename OT>
int embedding(const int64_t* tokens, int64_t n, const void* weight, int64_t V, int64_t D, int64_t stride, int masked,
              int64_t padding, float scale, void* out, hipStream_t s) {
  int lanes = 1;
  while (lanes < 64 && lanes * 8 < D) lanes *= 2;
  const int64_t most = ((int64_t)1 << 31) / lanes;  // rows of a launch, whose threads have to be fewer than 2^32
  for (int64_t at = 0; at < n; at += most) {
    const int64_t rows = n - at < most ? n - at : most;
    const unsigned blocks = (unsigned)cdiv(rows, 256 / lanes);
    const auto kernel = masked ? fl_embedding_kernel<WT, OT, true> : fl_embedding_kernel<WT, OT, false>;
    kernel<<<blocks, 256, 0, s>>>(tokens + at, rows, static_cast<const WT*>(weight), V, D, stride, lanes, padding, scale,
                                  static_cast<OT*>(out) + at * D);
    const int status = hip_status(hipGetLastError());
    if (status != FL_OK) return status;
  }
  return FL_OK;
}

static_assert(kMaxExtras * kJoinThreads < (int64_t)1 << 32 && (kMaxExtras + kMaxBuckets) * kSumThreads < (int64_t)1 << 32, "");

// how a call's tokens are sorted and summed
struct Plan {
  Sort s;
  int64_t extras;
  size_t counts, starts, extra, first, present, list, part, bytes;  // offsets
};

Plan plan_of(int64_t n, int64_t V, int64_t D) {
  Plan p = {};
  Sort& s = p.s;
  s.n = n;
  s.V = V;
  while (cdiv(V, (int64_t)1 << s.shift) > kMaxBuckets) ++s.shift;
  s.buckets = (int)cdiv(V, (int64_t)1 << s.shift);
  s.chunk = n <= kOneChunk ? kOneChunk : (int)(cdiv(cdiv(n, kMaxChunks), kSortThreads) * kSortThreads);
  s.chunks = (int)cdiv(n, s.chunk);
  if (s.chunks < 1) s.chunks = 1;
  const size_t row_bytes = (size_t)D * 4 << s.shift;
  const int64_t most = (int64_t)(kPartBytes / row_bytes) > 32 ? (int64_t)(kPartBytes / row_bytes) : 32;
  const int64_t least = std::max(cdiv(2 * n, most), cdiv(n, kMaxExtras));
  s.piece = (int)(cdiv(least, kPiece) * kPiece);
  if (s.piece < kPiece) s.piece = kPiece;
  p.extras = n / s.piece;  // (at most kMaxExtras)
  const auto take = [&](size_t bytes) {
    const size_t at = p.bytes;
    p.bytes += (bytes + 15) / 16 * 16;
    return at;
  };
  p.counts = take((size_t)s.chunks * kMaxBuckets * 4);
  p.starts = take((size_t)(s.buckets + 1) * 4);
  p.extra = take((size_t)(p.extras + 1) * 4);
  p.first = take((size_t)s.buckets * 4);
  p.present = take((size_t)p.extras * 2 * ((((size_t)1 << s.shift) + 31) / 32) * 4);
  p.list = take((size_t)n * sizeof(Entry));
  p.part = take((size_t)p.extras * 2 * row_bytes);
  return p;
}

template <typename GT, typename WT>
int embedding_grad(Plan p, const int64_t* tokens, const void* g, int64_t D, int64_t padding, float scale, void* out,
                   char* ws, hipStream_t stream) {
  Sort& s = p.s;
  s.tokens = tokens;
  s.padding = padding;
  s.counts = reinterpret_cast<uint32_t*>(ws + p.counts);
  s.starts = reinterpret_cast<uint32_t*>(ws + p.starts);
  s.extra = reinterpret_cast<uint32_t*>(ws + p.extra);
  s.first = reinterpret_cast<uint32_t*>(ws + p.first);
  s.present = reinterpret_cast<uint32_t*>(ws + p.present);
  s.list = reinterpret_cast<Entry*>(ws + p.list);
  if (s.chunks > 1) fl_embedding_count_kernel<<<(unsigned)s.chunks, kSortThreads, 0, stream>>>(s);
  fl_embedding_sort_kernel<<<(unsigned)s.chunks, kSortThreads, 0, stream>>>(s);
  fl_embedding_sum_kernel<GT, WT><<<(unsigned)(s.buckets + p.extras), kSumThreads, 0, stream>>>(
      s, (int)p.extras, static_cast<const GT*>(g), D, scale, reinterpret_cast<float*>(ws + p.part), static_cast<WT*>(out));
  if (p.extras) {
    constexpr int N = sizeof(GT) == 2 && sizeof(WT) == 2 ? 8 : 4;
    fl_embedding_join_kernel<N, WT><<<dim3((unsigned)p.extras, 4), kJoinThreads, 0, stream>>>(
        s, D, scale, reinterpret_cast<float*>(ws + p.part), static_cast<WT*>(out));
  }
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
  return sizes_ok(n, V, D) ? plan_of(n, V, D).bytes : 0;
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
  return call(plan_of(n, V, D), tokens, g, D, padding, scale, g_weight, static_cast<char*>(workspace), s);
}

}  // extern "C"
