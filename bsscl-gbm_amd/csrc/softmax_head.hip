// Softmax cross entropy of hidden x weight^T over a large vocabulary, and its
// gradient (the formulas stand in bsscl_hip.h).
//
// The counting rows are packed together first, so that rows without a label
// cost nothing and their values reach no sum.  A score exists only inside the
// tile that computes it: the tile leaves, per row, its maximum m_t and the sum
// of exp(z - m_t), and the row's lse follows from those of all tiles,
//   m = max m_t,   lse = m + log sum_t s_t exp(m_t - m).
// For the gradient a tile also leaves exp(z - m_t) (times the cap's slope) in
// the inputs' dtype: k_rows turns it into d loss / d score by one factor per
// row and tile, exp(m_t - m) / s times the row's weight, and puts the label's
// own value there from its float32 score, where p - 1 keeps what a rounded p
// would lose.  These rows of the vocabulary's length are made for a piece of
// the rows at a time (kPieceBytes; smaller calls are one piece, whose
// exponentials are rows x vocab in the inputs' dtype), and both products consume
// a piece before the next one takes its place.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "device_call.h"
#include "mfma_tile.h"

namespace bsscl {

namespace {

constexpr float kLog2E = 1.4426950408889634f;
constexpr int kRowPad = 256;    // rows of a piece: a multiple
constexpr int kColPad = 64;     // width of the packed rows: a multiple
constexpr int64_t kPieceBytes = int64_t(1) << 30;

struct HeadInfo {
  int32_t rows;      // counting rows
  float to_operand;  // what d loss / d score is multiplied by as an operand
  float from_operand;
  float lift;        // of the piece: its operands are divided by it as well
  int32_t low, high;  // in_order of the finite tile maxima so far (float16 with z-loss)
};

// Integers in the order of floats, its own inverse (for atomic minima and maxima).
__device__ __forceinline__ int32_t in_order(int32_t bits) {
  return bits ^ ((bits >> 31) & 0x7fffffff);
}

// Float16 operands hold 1 + 2 zeta lse up to 32 (63, with what the label's value
// adds); beyond that a power of two is divided out.  lse lies between the row's
// maximum, itself no lower than the lowest tile's, and the highest plus log of the
// classes, which is known before the piece's rows are scaled.
__device__ __forceinline__ float lift_of(const HeadInfo *info, float z_loss, float log_classes) {
  const float low = __builtin_bit_cast(float, in_order(info->low));
  const float high = __builtin_bit_cast(float, in_order(info->high));
  const float most = fmaxf(fabsf(1.f + 2.f * z_loss * low),
                           fabsf(1.f + 2.f * z_loss * (high + log_classes)));
  if (!(most > 32.f && most < INFINITY)) return 1.f;
  int e;
  (void)frexpf(most / 32.f, &e);
  return ldexpf(1.f, e);
}

// A tile's exponentials, at most 1, are kept times this: in float16 they would
// lose digits below 2^-14 of the tile's maximum otherwise.
template <typename T>
constexpr float kExpScale = std::is_same<T, _Float16>::value ? 32768.f : 1.f;

int64_t round_up(int64_t a, int64_t b) { return (a + b - 1) / b * b; }

// Rows of piece p of `pieces`, of the counting rows: equal parts, each a
// multiple of kRowPad, none longer than the host's piece.
struct Piece {
  int32_t begin, rows;
};
__device__ __forceinline__ Piece piece_of(int32_t n, int32_t p, int32_t pieces) {
  const int32_t each =
      (int32_t)((((int64_t)n + pieces - 1) / pieces + kRowPad - 1) / kRowPad * kRowPad);
  const int64_t begin = (int64_t)p * each;
  if (begin >= n) return {n, 0};
  return {(int32_t)begin, (int32_t)(n - begin < each ? n - begin : each)};
}

// Sum (largest) over the block's THREADS threads in a fixed order, in every one.
template <int THREADS, typename V, typename F>
__device__ __forceinline__ V block_fold(V v, V *tmp, F &&fold) {
  __syncthreads();
  tmp[threadIdx.x] = v;
  for (int k = THREADS / 2; k > 0; k >>= 1) {
    __syncthreads();
    if ((int)threadIdx.x < k) tmp[threadIdx.x] = fold(tmp[threadIdx.x], tmp[threadIdx.x + k]);
  }
  __syncthreads();
  return tmp[0];
}
template <int THREADS>
__device__ __forceinline__ double block_sum(double v, double *tmp) {
  return block_fold<THREADS>(v, tmp, [](double x, double y) { return x + y; });
}

__device__ __forceinline__ bool is_class(int64_t label, int32_t vocab) {
  return label >= 0 && label < vocab;
}

struct PrepareArgs {
  const int64_t *labels;
  const float *row_weight;
  int32_t rows, vocab, mean;
  float grad_scale;
  int32_t whole, narrow;  // float32, float16
  int32_t *idx, *lab;
  float *u;
  int32_t *pos;
  float *row_loss, *lse;
  HeadInfo *info;
};

// One block: the counting rows in order (idx, their labels and final weights),
// the place of each row (pos, -1 for none) and the zeros of the rows left out.
template <int THREADS>
__device__ void prepare(const PrepareArgs &a, double *tmp) {
  constexpr int kWaves = THREADS / 64;
  __shared__ int32_t wave_count[kWaves];
  const int tid = (int)threadIdx.x, lane = tid & 63, wid = tid >> 6;
  int32_t base = 0;
  double sum = 0.0, big = 0.0;
  for (int32_t at = 0; at < a.rows; at += THREADS) {
    const int32_t i = at + tid;
    const int64_t y = i < a.rows ? a.labels[i] : -1;
    const bool counts = is_class(y, a.vocab);
    const unsigned long long mask = __ballot(counts);
    if (lane == 0) wave_count[wid] = __popcll(mask);
    __syncthreads();
    int32_t before = base, all = 0;
    for (int w = 0; w < kWaves; ++w) {
      const int32_t c = wave_count[w];
      before += w < wid ? c : 0;
      all += c;
    }
    base += all;
    __syncthreads();
    if (i >= a.rows) continue;
    const int32_t p = before + __popcll(mask & ((1ull << lane) - 1));
    a.pos[i] = counts ? p : -1;
    if (counts) {
      const float w = a.row_weight ? a.row_weight[i] : 1.f;
      a.idx[p] = i;
      a.lab[p] = (int32_t)y;
      a.u[p] = w;
      sum += (double)w;
      big = fmax(big, fabs((double)w));
    } else {
      a.row_loss[i] = 0.f;
      a.lse[i] = 0.f;
    }
  }
  sum = block_sum<THREADS>(sum, tmp);
  big = block_fold<THREADS>(big, tmp, [](double x, double y) { return fmax(x, y); });
  const double share = a.mean ? (sum != 0.0 ? 1.0 / sum : 0.0) : 1.0;
  if (tid == 0) {
    // The largest weight becomes 1: rows of that weight (all rows, where none
    // are given) then have d loss / d label score at p - 1, which bf16 and
    // float16 hold to p for surprising labels, and not off by half a step like
    // any other multiple.  In float16 it becomes 2^10: a factor of 2^5 and more
    // is left to the largest value (1 + 2 zeta lse may exceed 1; lift_of), and
    // the smallest lies at 2^-35 of the weight.
    float m = (float)(big * fabs(share)) * fabsf(a.grad_scale);
    if (!(m >= 0x1p-100f && m <= 0x1p100f)) m = 1.f;
    const float one = a.narrow ? 1024.f : 1.f;
    a.info->rows = base;
    a.info->to_operand = a.whole ? 1.f : one / m;
    a.info->from_operand = a.whole ? 1.f : m / one;
    a.info->lift = 1.f;
    a.info->low = in_order(__builtin_bit_cast(int32_t, INFINITY));
    a.info->high = in_order(__builtin_bit_cast(int32_t, -INFINITY));
  }
  if (a.mean)
    for (int32_t p = tid; p < base; p += THREADS) a.u[p] = (float)((double)a.u[p] * share);
}

__global__ __launch_bounds__(1024) void k_head_prepare(const PrepareArgs a) {
  __shared__ double tmp[1024];
  prepare<1024>(a, tmp);
}

// Block b < rows: row b to its place among the counting rows, widened with
// zeros to `wide`, or zeros into d_hidden.  The kRowPad blocks after them: zero
// rows up to the next multiple of kRowPad.  Up to kCountRows rows a block counts
// its place itself, reading the labels before its own, and one block more does the
// work of k_head_prepare: a launch less (5 us of 57 at 128 x 512 x 4,099).  The
// kernels' own times, in one launch and in two: 3.4 and 6.6 us for 128 rows of 512,
// 5.5 and 7.9 for 1,024, 9.9 and 10.1 for 2,048, 20 and 15 for 4,096.
constexpr int kCountRows = 2048;

// Few rows of 16 bits with gradient stand twice among the packed rows, the second
// time from a row on that is told (0: once), and what rounding takes of d loss /
// d score stands beside the second ones: d_weight then sums both, and its operand
// has twice the digits.  A label's rounding would be most of its class's error
// otherwise: d_weight's was 1.6 times that of the rounded result at 1, 2 and 11
// rows, and is 1.0 to 1.05; beyond kTwiceRows, where labels' errors average, it is
// 1.1 to 1.4.  Kernel times with and without: 112 and 110 us (16 x 2,048 x 32,000
// bf16), 950 and 880 (64 x 4,096 x 131,072); 1,200 and 1,080 at 100 rows.
constexpr int kTwiceRows = 64;
static_assert(2 * kTwiceRows <= kRowPad && kTwiceRows % 32 == 0, "both fit what is packed anyway");
template <typename T>
__global__ __launch_bounds__(256) void k_pack_hidden(const T *hidden, int64_t stride,
                                                     int32_t width, int32_t wide,
                                                     const PrepareArgs a, T *packed,
                                                     int32_t again, T *d_hidden,
                                                     int64_t d_stride) {
  __shared__ double tmp[256];
  const int32_t b = (int32_t)blockIdx.x, rows = a.rows;
  if (b == rows + kRowPad) return prepare<256>(a, tmp);
  int32_t p;
  if (rows <= kCountRows) {
    int32_t n = 0;
    for (int32_t i = (int32_t)threadIdx.x; i < min(b, rows); i += 256)
      n += is_class(a.labels[i], a.vocab);
    p = (int32_t)block_sum<256>((double)n, tmp);
    if (b < rows && !is_class(a.labels[b], a.vocab)) p = -1;
  } else {
    p = b < rows ? a.pos[b] : a.info->rows;
  }
  if (b >= rows) {
    const int32_t n = p;
    p += b - rows;
    if (p >= (n + kRowPad - 1) / kRowPad * kRowPad) return;
    if (again && p >= again && p < again + n) return;
    for (int32_t d = (int32_t)threadIdx.x; d < wide; d += 256) packed[(int64_t)p * wide + d] = (T)0.f;
    return;
  }
  if (p >= 0) {
    const T *from = hidden + (int64_t)b * stride;
    for (int32_t d = (int32_t)threadIdx.x; d < wide; d += 256) {
      const T x = d < width ? from[d] : (T)0.f;
      packed[(int64_t)p * wide + d] = x;
      if (again) packed[(int64_t)(again + p) * wide + d] = x;
    }
  } else if (d_hidden) {
    for (int32_t d = (int32_t)threadIdx.x; d < width; d += 256)
      d_hidden[(int64_t)b * d_stride + d] = (T)0.f;
  }
}

// Tile `at` of slow x fast tiles: kGroup of the fast ones side by side, so that
// the tiles that run together share operands on both sides.
struct TileAt {
  int32_t slow, fast;
};
__device__ __forceinline__ TileAt tile_at(uint32_t at, uint32_t slow, uint32_t fast) {
  constexpr uint32_t kGroup = 8;
  const uint32_t group = at / (slow * kGroup), in = at % (slow * kGroup);
  const uint32_t width = min(kGroup, fast - group * kGroup);
  return {(int32_t)(in / width), (int32_t)(group * kGroup + in % width)};
}

// tanh(x): from 0.3 on as 1 - 2 / (1 + e^{2 |x|}), and below that the series,
// whose first term left out is 6e-8 of it.  Over all floats s from c / 10,000 to
// 20 c, c tanh_of(s / c) is off by at most 2.8 of 2^-24 c and 4.6e-7 of itself
// (c from 0.001 to 10,000): a cap far above the scores leaves them as they are.
// (tanhf makes the largest tile spill 56 registers, 3% of it without a cap too.)
__device__ __forceinline__ float tanh_of(float x) {
  const float e = __builtin_amdgcn_exp2f(fabsf(x) * (2.f * kLog2E)), q = x * x;
  float t = fmaf(q, 62.f / 2835.f, -17.f / 315.f);
  t = fmaf(q, t, 2.f / 15.f);
  t = fmaf(q, t, -1.f / 3.f);
  t = fmaf(q * x, t, x);
  return fabsf(x) < 0.3f ? t : copysignf(1.f - 2.f * __builtin_amdgcn_rcpf(1.f + e), x);
}

// Score tiles: BM classes x BN rows.  Label: int32 for packed rows, int64 for
// rows as the caller has them (info: none; `piece` rows).
//
// Classes are the m of the tile, so that a lane holds 4 MI classes of each of
// its rows and a row's maximum and sum take two lane exchanges and, where two
// waves share it, one through LDS.  With many rows the matrix cores are the
// bound (6,144 x 4,096 x 131,072 bf16 5.3 to 5.5 ms, 1.2 PFLOP/s with 1.6 GB of
// exponentials written).  A tile's start and end cost 10 us, with a cap 19, and
// writing the exponentials 1 to 16 more (1,536 rows x 32,768 classes bf16, three
// rounds of tiles: 22, 33, 60 and 122 us a round at widths 512 to 4,096, with
// exponentials 23, 49, 74 and 128).  With few rows the weight's bytes are the
// bound (1 x 2,048 x 32,000 bf16 22 us, 6 TB/s from the caches).
template <typename TL, typename Label>
__global__ __launch_bounds__(TL::kThreads) void k_scores(
    const typename TL::T *weight, int64_t w_stride, int32_t vocab, int32_t width,
    const typename TL::T *packed, int64_t wide, const Label *lab, const HeadInfo *info,
    int32_t piece, int32_t pieces, float softcap, int32_t tiles, float2 *stats, float *z_label,
    typename TL::T *P, int64_t ldp) {
  using T = typename TL::T;
  __shared__ __align__(1024) char lds[TL::kLdsOut];
  constexpr bool kPacked = sizeof(Label) == 4;
  Piece pc{0, piece};
  if constexpr (kPacked) pc = piece_of(info->rows, piece, pieces);
  const uint32_t row_tiles = (uint32_t)(pc.rows + TL::BN - 1) / TL::BN;
  const uint32_t total = row_tiles * (uint32_t)tiles;
  if (blockIdx.x >= total) return;
  const TileAt at = tile_at(xcd_order(blockIdx.x, total), (uint32_t)tiles, row_tiles);
  const int32_t v0 = at.slow * TL::BM, r0 = at.fast * TL::BN;
  typename TL::A a;
  typename TL::B b;
  a.init(weight, w_stride, v0, vocab);
  b.init(packed + pc.begin * wide, wide, r0,
         kPacked ? (pc.rows + kRowPad - 1) / kRowPad * kRowPad : pc.rows);
  Acc4 acc[TL::MI][TL::NI] = {};
  TL::walk(a, b, 0, width, lds, acc);

  const int wave = (int)threadIdx.x >> 6, l = (int)threadIdx.x & 63;
  const int wm = wave / TL::kWavesN * TL::WM, wn = wave % TL::kWavesN * TL::WN;
  // Everything up to the exponential is one instruction a score where it can
  // be: caps, classes beyond the vocabulary and labels are looked after by
  // branches that all lanes of a wave take together.
  auto each = [&](auto f) {
#pragma unroll
    for (int j = 0; j < TL::NI; ++j)
#pragma unroll
      for (int i = 0; i < TL::MI; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          acc[i][j][r] = f(acc[i][j][r], wm + i * 16 + (l >> 4) * 4 + r);
  };
  const float to_slope = softcap > 0.f ? 1.f / softcap : 0.f;
  if (softcap > 0.f) each([&](float z, int) { return softcap * tanh_of(z * to_slope); });
  if (v0 + TL::BM > vocab)
    each([&](float z, int v) { return v0 + v < vocab ? z : -INFINITY; });
  // A lane holds rows wn + 16 j + l % 16 and four classes of each 16; the lanes
  // of equal l % 16 and the waves along m share a row.
  float *part = reinterpret_cast<float *>(lds);  // [kWavesM][BN]
  float top[TL::NI];
#pragma unroll
  for (int j = 0; j < TL::NI; ++j) {
    const int n = wn + j * 16 + (l & 15);
    const Label y = (r0 + n < pc.rows ? lab[pc.begin + r0 + n] : -1) - v0 - wm;
    if (__any(y >= 0 && y < TL::WM)) {
#pragma unroll
      for (int i = 0; i < TL::MI; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (i * 16 + (l >> 4) * 4 + r == y) z_label[r0 + n] = acc[i][j][r];
    }
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < TL::MI; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) m = fmaxf(m, acc[i][j][r]);
    m = fmaxf(m, __shfl_xor(m, 16));
    top[j] = fmaxf(m, __shfl_xor(m, 32));
    if (TL::kWavesM > 1 && l < 16) part[wave / TL::kWavesN * TL::BN + n] = top[j];
  }
  if constexpr (TL::kWavesM > 1) {
    __syncthreads();
#pragma unroll
    for (int j = 0; j < TL::NI; ++j)
#pragma unroll
      for (int w = 0; w < TL::kWavesM; ++w)
        top[j] = fmaxf(top[j], part[w * TL::BN + wn + j * 16 + (l & 15)]);
    __syncthreads();
  }
#pragma unroll
  for (int j = 0; j < TL::NI; ++j) {
    // The difference first: the maximum's exponential is 1 whatever its size, so
    // that sums are at least 1 and no p exceeds 1.
    const float base = top[j] == -INFINITY ? 0.f : top[j];
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < TL::MI; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float z = acc[i][j][r], e = __builtin_amdgcn_exp2f((z - base) * kLog2E);
        s += e;
        if (!P) continue;
        if (softcap > 0.f) {
          const float t = e > 0.f ? z * to_slope : 0.f;
          acc[i][j][r] = e * (kExpScale<T> - kExpScale<T> * t * t);
        } else {
          acc[i][j][r] = e * kExpScale<T>;
        }
      }
    s += __shfl_xor(s, 16);
    s += __shfl_xor(s, 32);
    if (l < 16) part[wave / TL::kWavesN * TL::BN + wn + j * 16 + l] = s;
  }
  __syncthreads();
  if (wm == 0 && l < 16)
#pragma unroll
    for (int j = 0; j < TL::NI; ++j) {
      const int n = wn + j * 16 + l;
      float s = part[n];
      for (int w = 1; w < TL::kWavesM; ++w) s += part[w * TL::BN + n];
      if (r0 + n < pc.rows) stats[(int64_t)(r0 + n) * tiles + at.slow] = make_float2(top[j], s);
    }
  if (!P) return;
  __syncthreads();
  TL::stage_out(lds, [&](int i, int j, int r) { return (T)acc[i][j][r]; });
  __syncthreads();
  TL::read_out(lds, [&](int n, int m, Int4 x) {
    // (Past the caches, which keep the operands: 1% of the kernel.)
    __builtin_nontemporal_store(x,
                                reinterpret_cast<Int4 *>(P + (int64_t)(r0 + n) * ldp + v0 + m));
  });
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int k = 32; k > 0; k >>= 1) v = fmaxf(v, __shfl_xor(v, k));
  return v;
}
__device__ __forceinline__ float wave_add(float v) {
#pragma unroll
  for (int k = 32; k > 0; k >>= 1) v += __shfl_xor(v, k);
  return v;
}

// (m, s) with s exp(m) the sum over the tiles first, first + by, ...: rescaled
// as the maximum grows.  (A tile of maximum -inf holds no score above it: its sum
// is 0, or NaN, which stays.)
__device__ __forceinline__ float2 tiles_sum(const float2 *st, int32_t tiles, int32_t first,
                                            int32_t by) {
  float m = -INFINITY, s = 0.f;
#pragma unroll 4
  for (int32_t t = first; t < tiles; t += by) {
    const float2 x = st[t];
    if (x.x > m) {
      s = m == -INFINITY ? s + x.y : s * expf(m - x.x) + x.y;
      m = x.x;
    } else {
      s += x.x == -INFINITY ? x.y : x.y * expf(x.x - m);
    }
  }
  return make_float2(m, s);
}

// (m, s) of a row from its tiles' statistics: lse = m + log s.
__device__ __forceinline__ float lse_of(float2 x) {
  return (x.x == -INFINITY ? 0.f : x.x) + logf(x.y);
}
// The row's negative log-probability of its label, whose score is zy: the parts
// of lse apart, so that a loss far below lse keeps its digits and none is
// below 0 (zy is one of the scores, and s is at least 1).
__device__ __forceinline__ float minus_log_p(float2 x, float zy) {
  return ((x.x == -INFINITY ? 0.f : x.x) - zy) + logf(x.y);
}

// A row's (m, s) by the block's kRowThreads threads.
constexpr int kRowThreads = 256;
__device__ float2 row_sum(const float2 *st, int32_t tiles, float *red) {
  constexpr int kWaves = kRowThreads / 64;
  const int tid = (int)threadIdx.x, wid = tid >> 6;
  const float2 own = tiles_sum(st, tiles, tid, kRowThreads);
  const float m = own.x;
  float s = own.y;
  float top = wave_max(m);
  if ((tid & 63) == 0) red[wid] = top;
  __syncthreads();
  top = red[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) top = fmaxf(top, red[w]);
  s = wave_add(m == -INFINITY ? s : s * expf(m - top));
  if ((tid & 63) == 0) red[kWaves + wid] = s;
  __syncthreads();
  s = red[kWaves];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) s += red[kWaves + w];
  return make_float2(top, s);
}

// Up to kFewRows rows as the caller has them, one block: each wave takes a part
// of a row's tiles, and the rows' weighted sum follows in their order.
constexpr int kFewRows = 32;
__global__ __launch_bounds__(1024) void k_few_rows(const int64_t *labels, const float *row_weight,
                                                   int32_t rows, int32_t vocab, int32_t mean,
                                                   float z_loss, int32_t tiles,
                                                   const float2 *stats, const float *z_label,
                                                   float *loss, float *row_loss, float *lse_out) {
  constexpr int kWaves = 16;
  __shared__ float2 part[kFewRows][kWaves];
  __shared__ float value[kFewRows];
  const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
  const int parts = rows <= 1 ? 16 : rows <= 2 ? 8 : rows <= 4 ? 4 : rows <= 8 ? 2 : 1;
  for (int r = wave / parts; r < rows; r += kWaves / parts) {
    float2 x = tiles_sum(stats + (int64_t)r * tiles, tiles, wave % parts * 64 + lane, parts * 64);
    const float top = wave_max(x.x);
    x.y = wave_add(x.x == -INFINITY ? x.y : x.y * expf(x.x - top));
    if (lane == 0) part[r][wave % parts] = make_float2(top, x.y);
  }
  __syncthreads();
  const int r = (int)threadIdx.x;
  if (r < rows) {
    const float2 x = tiles_sum(part[r], parts, 0, 1);
    const float lse = lse_of(x);
    const int64_t y = labels[r];
    const bool counts = y >= 0 && y < vocab;
    const float l = counts ? minus_log_p(x, z_label[r]) + z_loss * lse * lse : 0.f;
    row_loss[r] = l;
    lse_out[r] = counts ? lse : 0.f;
    value[r] = l;
  }
  __syncthreads();
  if (threadIdx.x != 0) return;
  double s = 0.0, all = 0.0;
  for (int i = 0; i < rows; ++i) {
    if (labels[i] < 0 || labels[i] >= vocab) continue;
    const double w = row_weight ? row_weight[i] : 1.0;
    all += w;
    s += w * value[i];
  }
  *loss = (float)(!mean ? s : all != 0.0 ? s / all : 0.0);
}

// The range of a piece's finite tile maxima, joined to that of the pieces before
// it.  A pass of its own over what the tiles left, with one pair of atomics a
// block (7 us of 600 at 1,500 x 32,003; 15 with a pair a wave, and a pair at the
// end of each wave of a tile made the tiles take 55 us longer there).
constexpr int kRangeBlocks = 64;
__global__ __launch_bounds__(1024) void k_range(HeadInfo *info, int32_t piece, int32_t pieces,
                                                int32_t tiles, const float2 *stats) {
  __shared__ float tmp[1024];
  const int64_t n = (int64_t)piece_of(info->rows, piece, pieces).rows * tiles;
  float low = INFINITY, high = -INFINITY;
#pragma unroll 4
  for (int64_t i = (int64_t)blockIdx.x * 1024 + threadIdx.x; i < n; i += kRangeBlocks * 1024) {
    const float top = stats[i].x;
    const bool finite = fabsf(top) < INFINITY;
    low = fminf(low, finite ? top : INFINITY);
    high = fmaxf(high, finite ? top : -INFINITY);
  }
  low = block_fold<1024>(low, tmp, [](float x, float y) { return fminf(x, y); });
  high = block_fold<1024>(high, tmp, [](float x, float y) { return fmaxf(x, y); });
  if (threadIdx.x != 0) return;
  atomicMin(&info->low, in_order(__builtin_bit_cast(int32_t, low)));
  atomicMax(&info->high, in_order(__builtin_bit_cast(int32_t, high)));
}

// One block per row of the piece: lse and loss from the tiles' statistics;
// with P, the row of d loss / d score in its place.  Bound by memory with P: a
// block keeps kVecs 16-byte loads a thread in flight (6,144 x 131,072 bf16 read
// and written in 600 us, 5.4 TB/s; 645 us with loads that stay in the caches).
template <typename T>
__global__ __launch_bounds__(kRowThreads) void k_rows(
    HeadInfo *info, int32_t piece, int32_t pieces, const int32_t *idx, const int32_t *lab,
    const float *u, float softcap, float z_loss, float grad_scale, int32_t tiles, int32_t tile_v,
    const float2 *stats, const float *z_label, T *P, int64_t ldp, int32_t again,
    float *own_rest, float *row_loss, float *lse_out) {
  __shared__ float red[2 * kRowThreads / 64];
  constexpr int kVec = 16 / (int)sizeof(T), kVecs = 4;
  const Piece pc = piece_of(info->rows, piece, pieces);
  const int32_t r = (int32_t)blockIdx.x;
  const int tid = (int)threadIdx.x;
  Int4 *row = reinterpret_cast<Int4 *>(P + (int64_t)r * ldp);
  const int32_t n = (int32_t)(ldp / kVec);
  if (r >= pc.rows) {
    // The products read whole steps of rows: zeros behind the last one.
    if (again && r >= again && r < again + pc.rows) return;
    if (P && r < (pc.rows + kRowPad - 1) / kRowPad * kRowPad)
      for (int32_t i = tid; i < n; i += kRowThreads) row[i] = Int4{0, 0, 0, 0};
    return;
  }
  const float2 *st = stats + (int64_t)r * tiles;
  const float2 sum = row_sum(st, tiles, red);
  const int32_t c = pc.begin + r, y = lab[c];
  const float zy = z_label[r], lse = lse_of(sum), nll = minus_log_p(sum, zy);
  if (tid == 0) {
    row_loss[idx[c]] = nll + z_loss * lse * lse;
    lse_out[idx[c]] = lse;
  }
  if (!P) return;
  float lift = 1.f;
  if constexpr (std::is_same<T, _Float16>::value)
    if (z_loss > 0.f) {
      lift = lift_of(info, z_loss, logf((float)ldp));
      if (r == 0 && tid == 0) info->lift = lift;  // for the products
    }
  const float g = u[c] * grad_scale * (info->to_operand / lift), zl = 2.f * z_loss * lse;
  const float py = expm1f(-nll);
  const float slope = softcap > 0.f ? 1.f - (zy / softcap) * (zy / softcap) : 1.f;
  const float own = g * slope * (py + zl * (py + 1.f));
  // What rounding takes of the label's value, the row's largest as a rule:
  // k_d_hidden_sum adds it times the label's row of the weight.
  if (tid == 0) own_rest[r] = own - (float)(T)own;
  const float scale = g * (1.f + zl) / (kExpScale<T> * sum.y);
  Int4 *rest = again ? row + (int64_t)again * n : nullptr;
  const int tile_shift = 31 - __clz(tile_v / kVec);
  for (int32_t i0 = tid; i0 < n; i0 += kRowThreads * kVecs) {
    Int4 x[kVecs];
    float f[kVecs];
#pragma unroll
    for (int k = 0; k < kVecs; ++k) {
      const int32_t i = i0 + k * kRowThreads;
      if (i < n) {
        x[k] = __builtin_nontemporal_load(row + i);
        f[k] = st[i >> tile_shift].x;
      }
    }
#pragma unroll
    for (int k = 0; k < kVecs; ++k) {
      const int32_t i = i0 + k * kRowThreads;
      if (i >= n) continue;
      const float by = expf(f[k] - sum.x) * scale;
      typedef T TV __attribute__((ext_vector_type(kVec)));
      TV v = __builtin_bit_cast(TV, x[k]), low;
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        const float d = i * kVec + e == y ? own : (float)v[e] * by;
        v[e] = (T)d;
        low[e] = (T)(d - (float)v[e]);
      }
      row[i] = __builtin_bit_cast(Int4, v);
      if (rest) rest[i] = __builtin_bit_cast(Int4, low);
    }
  }
}

// What the two products of a piece take.
struct ProductArgs {
  const void *P;
  int64_t ldp;
  const void *packed;
  int32_t wide, vocab, width;
  const HeadInfo *info;
  int32_t piece, pieces;
  // d_hidden: the weight (w_width columns), its vocabulary in `splits` parts
  const void *weight;
  int64_t w_stride;
  int32_t w_width, splits, split_v;
  float *part;
  int64_t part_stride;
  // d_weight
  float *sum;
  void *d_weight;
  int64_t dw_stride;
  int32_t dw_vec, again;
};

// d_hidden of a piece: BM columns x BN rows over a part of the vocabulary, as
// float32 sums of their own.  Tile `block` of those there are.
template <typename TL>
__device__ __forceinline__ void d_hidden_tile(const ProductArgs &g, uint32_t block, char *lds) {
  using T = typename TL::T;
  const T *P = static_cast<const T *>(g.P), *weight = static_cast<const T *>(g.weight);
  const Piece pc = piece_of(g.info->rows, g.piece, g.pieces);
  const uint32_t row_tiles = (uint32_t)(pc.rows + TL::BN - 1) / TL::BN;
  const uint32_t col_tiles = (uint32_t)(g.w_width + TL::BM - 1) / TL::BM;
  const uint32_t each = row_tiles * col_tiles, total = each * (uint32_t)g.splits;
  if (block >= total) return;
  const uint32_t idx = xcd_order(block, total);
  const TileAt at = tile_at(idx % each, col_tiles, row_tiles);
  const int32_t d0 = at.slow * TL::BM, r0 = at.fast * TL::BN, split = (int32_t)(idx / each);
  typename TL::A a;
  typename TL::B b;
  a.init(weight, g.w_stride, d0, g.w_width);
  b.init(P, g.ldp, r0, (pc.rows + kRowPad - 1) / kRowPad * kRowPad);
  Acc4 acc[TL::MI][TL::NI] = {};
  TL::walk(a, b, (int64_t)split * g.split_v,
           min((int64_t)(split + 1) * g.split_v, (int64_t)g.vocab), lds, acc);
  const int wave = (int)threadIdx.x >> 6, l = (int)threadIdx.x & 63;
  const int wm = wave / TL::kWavesN * TL::WM, wn = wave % TL::kWavesN * TL::WN;
#pragma unroll
  for (int j = 0; j < TL::NI; ++j) {
    const int32_t r = r0 + wn + j * 16 + (l & 15);
    if (r >= pc.rows) continue;
    float *out = g.part + (int64_t)split * g.part_stride + (int64_t)r * g.wide;
#pragma unroll
    for (int i = 0; i < TL::MI; ++i) {
      const int32_t d = d0 + wm + i * 16 + (l >> 4) * 4;
      if (d < g.wide) *reinterpret_cast<Acc4 *>(out + d) = acc[i][j];
    }
  }
}

// d_weight of a piece: BM columns x BN classes over the piece's rows; pieces
// before the last add up in float32.  Tile `block` of `blocks`.
template <typename TL>
__device__ __forceinline__ void d_weight_tile(const ProductArgs &g, uint32_t block,
                                              uint32_t blocks, char *lds) {
  using T = typename TL::T;
  T *d_weight = static_cast<T *>(g.d_weight);
  const int32_t wide = g.wide, vocab = g.vocab, width = g.width, piece = g.piece,
                pieces = g.pieces;
  const Piece pc = piece_of(g.info->rows, piece, pieces);
  const uint32_t col_tiles = (uint32_t)(width + TL::BM - 1) / TL::BM;
  const uint32_t v_tiles = (uint32_t)(vocab + TL::BN - 1) / TL::BN;
  const TileAt at = tile_at(xcd_order(block, blocks), v_tiles, col_tiles);
  const int32_t v0 = at.slow * TL::BN, d0 = at.fast * TL::BM;
  typename TL::A a;
  typename TL::B b;
  a.init(static_cast<const T *>(g.packed) + (int64_t)pc.begin * wide, wide, d0, wide);
  b.init(static_cast<const T *>(g.P), g.ldp, v0, (int32_t)g.ldp);
  Acc4 acc[TL::MI][TL::NI] = {};
  const int32_t rows = pc.rows ? g.again + pc.rows : 0;
  TL::walk(a, b, 0, (rows + TL::kStep - 1) / TL::kStep * TL::kStep, lds, acc);
  const float lift = g.info->lift;
  if (pieces > 1) {
    const int wave = (int)threadIdx.x >> 6, l = (int)threadIdx.x & 63;
    const int wm = wave / TL::kWavesN * TL::WM, wn = wave % TL::kWavesN * TL::WN;
#pragma unroll
    for (int j = 0; j < TL::NI; ++j) {
      const int32_t v = v0 + wn + j * 16 + (l & 15);
      if (v >= vocab) continue;
#pragma unroll
      for (int i = 0; i < TL::MI; ++i) {
        const int32_t d = d0 + wm + i * 16 + (l >> 4) * 4;
        if (d >= wide) continue;
        Acc4 *p = reinterpret_cast<Acc4 *>(g.sum + (int64_t)v * wide + d);
        acc[i][j] *= lift;
        if (piece > 0) acc[i][j] += *p;
        if (piece < pieces - 1) *p = acc[i][j];
      }
    }
    if (piece < pieces - 1) return;
  }
  const float back = pieces > 1 ? g.info->from_operand : g.info->from_operand * lift;
  TL::stage_out(lds, [&](int i, int j, int r) { return (T)(acc[i][j][r] * back); });
  __syncthreads();
  if (g.dw_vec) {
    TL::read_out(lds, [&](int n, int m, Int4 x) {
      if (v0 + n < vocab && d0 + m < width)
        *reinterpret_cast<Int4 *>(d_weight + (int64_t)(v0 + n) * g.dw_stride + d0 + m) = x;
    });
  } else {
    TL::read_out_one(lds, [&](int n, int m, T x) {
      if (v0 + n < vocab && d0 + m < width) d_weight[(int64_t)(v0 + n) * g.dw_stride + d0 + m] = x;
    });
  }
}

template <typename TL>
__global__ __launch_bounds__(TL::kThreads) void k_d_hidden(const ProductArgs g) {
  __shared__ __align__(1024) char lds[TL::kLds];
  d_hidden_tile<TL>(g, blockIdx.x, lds);
}
template <typename TL>
__global__ __launch_bounds__(TL::kThreads) void k_d_weight(const ProductArgs g) {
  __shared__ __align__(1024) char lds[TL::kLdsOut];
  d_weight_tile<TL>(g, blockIdx.x, gridDim.x, lds);
}
// Both in one launch, d_hidden's long tiles (`hidden` blocks, a multiple of 8)
// first: d_weight's short ones fill the CUs that they leave (1,500 x 2,048 x
// 32,003 fp16 422 us, 501 in two launches; 6,144 x 4,096 x 131,072 bf16 10.1 to
// 10.5 ms, 1.3 PFLOP/s, the same in two).
template <typename TH, typename TW>
__global__ __launch_bounds__(TH::kThreads) void k_products(const ProductArgs g, uint32_t hidden) {
  static_assert(TH::kThreads == TW::kThreads);
  __shared__ __align__(1024) char lds[TH::kLds > TW::kLdsOut ? TH::kLds : TW::kLdsOut];
  if (blockIdx.x < hidden)
    d_hidden_tile<TH>(g, blockIdx.x, lds);
  else
    d_weight_tile<TW>(g, blockIdx.x - hidden, gridDim.x - hidden, lds);
}

// loss = sum of u * row_loss over the counting rows, in their order.
struct LossArgs {
  const HeadInfo *info;
  const int32_t *idx;
  const float *u, *row_loss;
  float *loss;
};
template <int THREADS>
__device__ void loss_sum(const LossArgs &a, double *tmp) {
  double s = 0.0;
  for (int32_t p = (int32_t)threadIdx.x; p < a.info->rows; p += THREADS)
    s += (double)a.u[p] * (double)a.row_loss[a.idx[p]];
  s = block_sum<THREADS>(s, tmp);
  if (threadIdx.x == 0) *a.loss = (float)s;
}

__global__ __launch_bounds__(1024) void k_loss_sum(const LossArgs a) {
  __shared__ double tmp[1024];
  loss_sum<1024>(a, tmp);
}

// The parts of d_hidden added up in their order, into the rows' places, with
// what rounding took of the label's value; block 0 adds up the loss (of the last
// piece, when all rows have theirs).
template <typename T>
__global__ __launch_bounds__(256) void k_d_hidden_sum(
    int32_t piece, int32_t pieces, const LossArgs loss, int32_t splits, const float *part,
    int64_t part_stride, int32_t wide, int32_t width, const int32_t *lab, const float *own_rest,
    const T *weight, int64_t w_stride, T *d_hidden, int64_t d_stride, int32_t vec) {
  __shared__ double tmp[256];
  if (blockIdx.x == 0) {
    if (piece == pieces - 1) loss_sum<256>(loss, tmp);
    return;
  }
  const HeadInfo *info = loss.info;
  const Piece pc = piece_of(info->rows, piece, pieces);
  const int32_t r = (int32_t)blockIdx.x - 1;
  if (r >= pc.rows) return;
  const float back = info->from_operand * info->lift;
  T *row = d_hidden + (int64_t)loss.idx[pc.begin + r] * d_stride;
  const T *own_row = weight + (int64_t)lab[pc.begin + r] * w_stride;
  const float rest = own_rest[r];
  typedef T T4 __attribute__((ext_vector_type(4)));
  for (int32_t d = (int32_t)threadIdx.x * 4; d < width; d += 1024) {
    const float *p = part + (int64_t)r * wide + d;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    if (rest != 0.f) {
      const T4 w = *reinterpret_cast<const T4 *>(own_row + d);
      s = make_float4(rest * (float)w[0], rest * (float)w[1], rest * (float)w[2],
                      rest * (float)w[3]);
    }
#pragma unroll 4
    for (int32_t k = 0; k < splits; ++k) {
      const float4 x = *reinterpret_cast<const float4 *>(p + (int64_t)k * part_stride);
      s = make_float4(s.x + x.x, s.y + x.y, s.z + x.z, s.w + x.w);
    }
    const T4 v = {(T)(s.x * back), (T)(s.y * back), (T)(s.z * back), (T)(s.w * back)};
    if (vec && d + 4 <= width) {
      *reinterpret_cast<T4 *>(row + d) = v;
      continue;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (d + e < width) row[d + e] = v[e];
  }
}

// Rows of the weight at a stride and width that the tiles can load from: a
// thread gathers 16 bytes of a row.
template <typename T>
__global__ __launch_bounds__(256) void k_pack_weight(const T *weight, int64_t stride,
                                                     int32_t vocab, int32_t width, int32_t wide,
                                                     T *packed) {
  constexpr int N = 16 / (int)sizeof(T);
  typedef T TV __attribute__((ext_vector_type(N)));
  const uint32_t chunks = (uint32_t)wide / N;
  for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;; e += (int64_t)gridDim.x * 256) {
    const int64_t v = e / chunks;
    if (v >= vocab) return;
    const int32_t d = (int32_t)(e - v * chunks) * N;
    const T *from = weight + v * stride + d;
    TV x;
#pragma unroll
    for (int k = 0; k < N; ++k) x[k] = d + k < width ? from[k] : (T)0.f;
    *reinterpret_cast<TV *>(packed + e * N) = x;
  }
}

// The tile shapes: 256 x 256 fills the matrix cores best and needs a whole
// CU's LDS; three of 128 x 64 share a CU (128 x 128 takes 461 us where it takes
// 424, 700 x 1,024 x 30,011 float32: fewer rows are padding, and the last round
// is shorter); 128 x 32 wastes less where there are few rows.
enum Shape : int32_t { kBig, kMid, kThin };
template <typename T, Shape S, bool A_ACROSS, bool B_ACROSS>
using TileOf = std::conditional_t<
    S == kBig, Tile<T, 256, 256, 128, 64, A_ACROSS, B_ACROSS, 128, 2>,
    std::conditional_t<S == kMid, Tile<T, 128, 64, 64, 32, A_ACROSS, B_ACROSS, 128, 2>,
                       Tile<T, 128, 32, 32, 32, A_ACROSS, B_ACROSS, 128, 3>>>;
constexpr int shape_m(Shape s) { return s == kBig ? 256 : 128; }
constexpr int shape_n(Shape s) { return s == kBig ? 256 : s == kMid ? 64 : 32; }

int64_t tiles_of(Shape s, int64_t m, int64_t n) {
  return ((m + shape_m(s) - 1) / shape_m(s)) * ((n + shape_n(s) - 1) / shape_n(s));
}

constexpr int64_t kCus = 256;

// Where a call's intermediate values lie in its workspace.
struct HeadPlan {
  int32_t rows, width, wide, vocab, tiles, tile_v;
  int32_t piece_rows, pieces, splits, split_v;
  Shape scores, d_hidden, d_weight;
  bool pack_weight;
  int64_t ldp;
  size_t info, idx, lab, u, pos, packed, stats, z_label, own_rest, P, part, sum, weight, bytes;
};

// Grids stay below 2^32 threads, and what a tile loads within 2^31 bytes.
constexpr int64_t kMostRows = 8000000, kMostVocab = 4000000, kMostWidth = 65536;
constexpr int64_t kMostPiece = 1 << 20;

int head_plan(int32_t dtype, int64_t rows, int64_t width, int64_t vocab, const void *weight,
              int64_t w_stride, bool grad, HeadPlan *pl) {
  if (dtype != BSSCL_BF16 && dtype != BSSCL_F16 && dtype != BSSCL_F32)
    return set_error(BSSCL_EINVAL, "softmax head: unknown dtype " + std::to_string(dtype));
  if (rows < 1 || vocab < 1 || width < 1 || rows > kMostRows || vocab > kMostVocab ||
      width > kMostWidth)
    return set_error(BSSCL_EINVAL,
                     "softmax head: rows must be in [1, 8000000], vocab in [1, 4000000], width in "
                     "[1, 65536]");
  const bool f32 = dtype == BSSCL_F32;
  const int64_t es = f32 ? 4 : 2;
  HeadPlan p{};
  p.rows = (int32_t)rows;
  p.width = (int32_t)width;
  p.wide = (int32_t)round_up(width, kColPad);
  p.vocab = (int32_t)vocab;
  // The largest tile that gives every other CU one and whose rows are not for
  // the most part padding.  Measured (us, kBig against kMid): scores of 64 rows x
  // 4,096 x 131,072 bf16 308 and 248, of 256 rows 293 and 475, of 512 rows x
  // 2,048 x 32,000 (250 tiles) 70 and 115; d_weight of 16 rows x 2,048 x 32,000 38
  // and 44, of 1,500 rows 187 and 291; kMid against kThin: scores of 700 x 1,024 x
  // 30,011 float32 425 and 474, of 128 x 512 x 4,099 (66 tiles) 29 and 18.
  auto shape = [&](int64_t m, int64_t n) {
    if (!f32 && n > 128 && tiles_of(kBig, m, n) >= kCus / 2) return kBig;
    return n > 32 && tiles_of(kMid, m, n) >= kCus / 2 ? kMid : kThin;
  };
  p.scores = shape(vocab, rows);
  p.tile_v = shape_m(p.scores);
  p.tiles = (int32_t)((vocab + p.tile_v - 1) / p.tile_v);
  p.ldp = (int64_t)p.tiles * p.tile_v;
  const int64_t row_bytes = grad ? p.ldp * es : (int64_t)p.tiles * (int64_t)sizeof(float2);
  // One piece takes no float32 sums of d_weight: it may have their room.
  const int64_t one = grad ? kPieceBytes + vocab * p.wide * 4 : kPieceBytes;
  const int64_t all = round_up(rows, kRowPad);
  const int64_t fit =
      all * row_bytes <= one && all <= kMostPiece
          ? all
          : std::max<int64_t>(kRowPad, kPieceBytes / row_bytes / kRowPad * kRowPad);
  p.piece_rows = (int32_t)std::min({fit, all, kMostPiece});
  p.pieces = (int32_t)((rows + p.piece_rows - 1) / p.piece_rows);
  if (grad) {
    const int64_t piece = std::min<int64_t>(rows, p.piece_rows);
    p.d_hidden = piece <= 32 ? kThin : !f32 && width >= 256 && piece >= 256 ? kBig : kMid;
    if (p.d_hidden == kMid && tiles_of(kMid, width, piece) < kCus / 16) p.d_hidden = kThin;
    p.d_weight = shape(width, vocab);
    // d_hidden's sums run over the whole vocabulary, in parts that fill the CUs.
    // The times here are estimates in microseconds; what they lead to, against half
    // and twice the parts (products and sums of parts): 423 (468, 454) at 1,500 x
    // 2,048 x 32,003 fp16, 474 (438, 508) at 2,047 x 1,001 x 50,257 bf16, 50 (83, 69)
    // at 4,096 x 1,024 x 3,000 bf16, 37 (47, 34) at 2,048 x 512 x 4,099 bf16; d_hidden
    // alone 261 (225, 305) at 64 x 4,096 x 131,072 bf16, 32 (28, 42) at 16 x 2,048 x
    // 32,000 bf16, 1,570 (1,570, 1,610) at 1,024 x 2,048 x 50,257 float32.
    const int64_t step = 128 / es, steps = (vocab + step - 1) / step;
    const int64_t tiles = tiles_of(p.d_hidden, width, piece);
    const int64_t most = std::min<int64_t>(64, std::max<int64_t>(1, steps / 4));
    if (p.d_hidden == kBig && p.d_weight == kBig) {
      // One launch with d_weight's tiles behind: as few parts as make a tile
      // take half of the whole at most.
      const double step_us = 1.45, whole =
          (double)(tiles * steps) * step_us +
          (double)tiles_of(kBig, width, vocab) * ((double)(piece + 63) / 64 * step_us + 10.0);
      const double longest = 0.5 * whole / kCus;
      p.splits = (int32_t)std::min<int64_t>(
          most, std::max<int64_t>(1, (int64_t)std::ceil((double)steps * step_us / longest)));
    } else {
      // What a number of parts costs: rounds of tiles (a CU holds three kMid or
      // two kThin), each with a start and an end, and the parts' sums written and
      // read.  How many rows count is not known here: the mean over half, three
      // quarters and all.
      const int64_t at_once = (p.d_hidden == kBig ? 1 : p.d_hidden == kMid ? 3 : 2) * kCus;
      const double step_us =
          (f32 ? 8.0 : 1.0) * (p.d_hidden == kBig ? 1.4 : p.d_hidden == kMid ? 0.6 : 0.3);
      const double part_us = (double)piece * p.wide * 8 / 4e6;
      double best = 0.0;
      for (int64_t n = 1; n <= most; ++n) {
        double rounds = 0.0;
        for (int64_t share = 2; share <= 4; ++share)
          rounds += (double)((tiles * share / 4 * n + at_once - 1) / at_once) * 4 / share / 3;
        const double us =
            rounds * ((double)((steps + n - 1) / n) * step_us + 6.0) + (double)n * part_us;
        if (n == 1 || us < best) {
          best = us;
          p.splits = (int32_t)n;
        }
      }
    }
    p.split_v = (int32_t)((steps + p.splits - 1) / p.splits * step);
    p.splits = (int32_t)((vocab + p.split_v - 1) / p.split_v);
  }
  // Loads are of 16 bytes, within 2^31 bytes of a tile's first row.
  p.pack_weight = ((uintptr_t)weight & 15) || w_stride * es % 16 || width * es % 16 ||
                  w_stride * es * 256 >= (int64_t(1) << 31);
  size_t at = 0;
  auto take = [&](int64_t bytes) {
    const size_t here = at;
    at += (size_t)round_up(bytes, 256);
    return here;
  };
  p.info = take(sizeof(HeadInfo));
  p.idx = take(rows * 4);
  p.lab = take(rows * 4);
  p.u = take(rows * 4);
  p.pos = take(rows * 4);
  p.packed = take(round_up(rows, kRowPad) * p.wide * es);
  p.stats = take((int64_t)p.piece_rows * p.tiles * (int64_t)sizeof(float2));
  p.z_label = take((int64_t)p.piece_rows * 4);
  p.own_rest = take(grad ? (int64_t)p.piece_rows * 4 : 0);
  p.P = take(grad ? (int64_t)p.piece_rows * p.ldp * es : 0);
  p.part = take(grad ? (int64_t)p.splits * p.piece_rows * p.wide * 4 : 0);
  p.sum = take(grad && p.pieces > 1 ? vocab * p.wide * 4 : 0);
  p.weight = take(p.pack_weight ? vocab * p.wide * es : 0);
  p.bytes = at;
  *pl = p;
  return BSSCL_OK;
}

struct HeadCall {
  const void *hidden, *weight;
  int64_t h_stride, w_stride;
  const int64_t *labels;
  const float *row_weight;
  bool mean, grad;
  float softcap, z_loss, grad_scale;
  float *loss, *row_loss, *lse;
  void *d_hidden, *d_weight;
  int64_t dh_stride, dw_stride;
  char *ws;
};

// f(std::integral_constant<Shape, s>) for s; float32 has no 256 x 256 tile
// (its output would not fit LDS).
template <typename T, typename F>
void by_shape(Shape s, F &&f) {
  if constexpr (sizeof(T) == 2)
    if (s == kBig) return f(std::integral_constant<Shape, kBig>());
  if (s == kThin) return f(std::integral_constant<Shape, kThin>());
  f(std::integral_constant<Shape, kMid>());
}

int launched() {
  const hipError_t e = hipGetLastError();
  if (e == hipSuccess) return BSSCL_OK;
  return set_error(BSSCL_EDEVICE, std::string("softmax head: ") + hipGetErrorString(e));
}

template <typename T>
int run_head(hipStream_t st, const HeadPlan &p, const HeadCall &c) {
  auto *info = reinterpret_cast<HeadInfo *>(c.ws + p.info);
  auto *idx = reinterpret_cast<int32_t *>(c.ws + p.idx);
  auto *lab = reinterpret_cast<int32_t *>(c.ws + p.lab);
  auto *u = reinterpret_cast<float *>(c.ws + p.u);
  auto *pos = reinterpret_cast<int32_t *>(c.ws + p.pos);
  auto *packed = reinterpret_cast<T *>(c.ws + p.packed);
  auto *stats = reinterpret_cast<float2 *>(c.ws + p.stats);
  auto *z_label = reinterpret_cast<float *>(c.ws + p.z_label);
  auto *own_rest = reinterpret_cast<float *>(c.ws + p.own_rest);
  auto *P = c.grad ? reinterpret_cast<T *>(c.ws + p.P) : nullptr;
  auto *part = reinterpret_cast<float *>(c.ws + p.part);
  auto *sum = reinterpret_cast<float *>(c.ws + p.sum);
  auto *weight = static_cast<const T *>(c.weight);
  int64_t w_stride = c.w_stride;
  int32_t w_width = p.width;
  constexpr int64_t kSize = (int64_t)sizeof(T);
  // A few rows to be scored, where the tiles can load them: two launches.
  if (!c.grad && p.rows <= kFewRows && !p.pack_weight && ((uintptr_t)c.hidden & 15) == 0 &&
      (p.rows == 1 || (c.h_stride * kSize % 16 == 0 &&
                       c.h_stride * kSize * kFewRows < (int64_t(1) << 31)))) {
    using TL = TileOf<T, kThin, false, false>;
    k_scores<TL, int64_t><<<(unsigned)p.tiles, TL::kThreads, 0, st>>>(
        weight, w_stride, p.vocab, p.width, static_cast<const T *>(c.hidden),
        p.rows == 1 ? p.width : c.h_stride, c.labels, nullptr, p.rows, 1, c.softcap, p.tiles, stats,
        z_label, nullptr, 0);
    k_few_rows<<<1, 1024, 0, st>>>(c.labels, c.row_weight, p.rows, p.vocab, c.mean, c.z_loss,
                                   p.tiles, stats, z_label, c.loss, c.row_loss, c.lse);
    return launched();
  }
  if (p.pack_weight) {
    auto *w = reinterpret_cast<T *>(c.ws + p.weight);
    const int64_t chunks = (int64_t)p.vocab * p.wide * (int64_t)sizeof(T) / 16;
    k_pack_weight<T><<<(unsigned)std::min<int64_t>((chunks + 255) / 256, 1 << 20), 256, 0, st>>>(
        weight, w_stride, p.vocab, p.width, p.wide, w);
    weight = w;
    w_stride = w_width = p.wide;
  }
  const PrepareArgs prep{c.labels, c.row_weight, p.rows, p.vocab, c.mean, c.grad_scale,
                         sizeof(T) == 4, std::is_same<T, _Float16>::value, idx, lab, u, pos,
                         c.row_loss, c.lse, info};
  const bool count = p.rows <= kCountRows;
  const int32_t again =
      c.grad && sizeof(T) == 2 && p.rows <= kTwiceRows ? (int32_t)round_up(p.rows, 32) : 0;
  if (!count) k_head_prepare<<<1, 1024, 0, st>>>(prep);
  k_pack_hidden<T><<<(unsigned)p.rows + kRowPad + (count ? 1 : 0), 256, 0, st>>>(
      static_cast<const T *>(c.hidden), c.h_stride, p.width, p.wide, prep, packed, again,
      static_cast<T *>(c.d_hidden), c.dh_stride);
  const LossArgs loss{info, idx, u, c.row_loss, c.loss};
  const int64_t piece = std::min<int64_t>(p.rows, p.piece_rows);
  const int64_t part_stride = (int64_t)p.piece_rows * p.wide;
  const int dw_vec = ((uintptr_t)c.d_weight & 15) == 0 && c.dw_stride * kSize % 16 == 0 &&
                     p.width * kSize % 16 == 0;
  const int dh_vec =
      (uintptr_t)c.d_hidden % (4 * sizeof(T)) == 0 && c.dh_stride % 4 == 0;
  for (int32_t k = 0; k < p.pieces; ++k) {
    by_shape<T>(p.scores, [&](auto s) {
      using TL = TileOf<T, decltype(s)::value, false, false>;
      k_scores<TL, int32_t><<<(unsigned)tiles_of(s, p.vocab, piece), TL::kThreads, 0, st>>>(
          weight, w_stride, p.vocab, w_width, packed, p.wide, lab, info, k, p.pieces, c.softcap,
          p.tiles, stats, z_label, P, p.ldp);
    });
    if constexpr (std::is_same<T, _Float16>::value)
      if (c.grad && c.z_loss > 0.f)
        k_range<<<kRangeBlocks, 1024, 0, st>>>(info, k, p.pieces, p.tiles, stats);
    k_rows<T><<<(unsigned)(c.grad ? p.piece_rows : piece), kRowThreads, 0, st>>>(
        info, k, p.pieces, idx, lab, u, c.softcap, c.z_loss, c.grad_scale, p.tiles, p.tile_v, stats,
        z_label, P, p.ldp, again, own_rest, c.row_loss, c.lse);
    if (!c.grad) continue;
    const ProductArgs g{P, p.ldp, packed, p.wide, p.vocab, p.width, info, k, p.pieces, weight,
                        w_stride, w_width, p.splits, p.split_v, part, part_stride, sum, c.d_weight,
                        c.dw_stride, dw_vec, again};
    const unsigned hidden = (unsigned)(tiles_of(p.d_hidden, w_width, piece) * p.splits);
    const unsigned weights = (unsigned)tiles_of(p.d_weight, p.width, p.vocab);
    bool both = false;
    if constexpr (sizeof(T) == 2)
      if (p.d_hidden == kBig && p.d_weight == kBig) {
        using TH = TileOf<T, kBig, true, false>;
        using TW = TileOf<T, kBig, true, true>;
        const unsigned first = (hidden + 7) / 8 * 8;
        k_products<TH, TW><<<first + weights, TH::kThreads, 0, st>>>(g, first);
        both = true;
      }
    if (!both) {
      by_shape<T>(p.d_hidden, [&](auto s) {
        using TL = TileOf<T, decltype(s)::value, true, false>;
        k_d_hidden<TL><<<hidden, TL::kThreads, 0, st>>>(g);
      });
      by_shape<T>(p.d_weight, [&](auto s) {
        using TL = TileOf<T, decltype(s)::value, true, true>;
        k_d_weight<TL><<<weights, TL::kThreads, 0, st>>>(g);
      });
    }
    k_d_hidden_sum<T><<<(unsigned)piece + 1, 256, 0, st>>>(
        k, p.pieces, loss, p.splits, part, part_stride, p.wide, p.width, lab, own_rest, weight,
        w_stride, static_cast<T *>(c.d_hidden), c.dh_stride, dh_vec);
  }
  if (!c.grad) k_loss_sum<<<1, 1024, 0, st>>>(loss);
  return launched();
}

int head(int32_t device, void *stream, int32_t dtype, int64_t rows, int64_t width, int64_t vocab,
         int32_t reduction, int64_t workspace_bytes, const HeadCall &c) {
  HeadPlan p;
  const int rc = head_plan(dtype, rows, width, vocab, c.weight, c.w_stride, c.grad, &p);
  if (rc != BSSCL_OK) return rc;
  if (!c.hidden || !c.weight || !c.labels || !c.loss || !c.row_loss || !c.lse || !c.ws ||
      (c.grad && (!c.d_hidden || !c.d_weight)))
    return set_error(BSSCL_EINVAL, "softmax head: null argument");
  if (c.h_stride < width || c.w_stride < width ||
      (c.grad && (c.dh_stride < width || c.dw_stride < width)))
    return set_error(BSSCL_EINVAL, "softmax head: a row stride is below the width");
  if (reduction != BSSCL_SUM && reduction != BSSCL_MEAN)
    return set_error(BSSCL_EINVAL, "softmax head: unknown reduction");
  if (!(c.softcap == 0.f || (c.softcap >= 1e-6f && std::isfinite(c.softcap))))
    return set_error(BSSCL_EINVAL, "softmax head: softcap must be 0 or finite and >= 1e-6");
  if (!(c.z_loss >= 0.f) || !std::isfinite(c.z_loss) || !std::isfinite(c.grad_scale))
    return set_error(BSSCL_EINVAL,
                     "softmax head: z_loss must be finite and >= 0, grad_scale finite");
  if ((size_t)workspace_bytes < p.bytes || ((uintptr_t)c.ws & 255))
    return set_error(BSSCL_EINVAL, "softmax head: the workspace holds " +
                                       std::to_string(workspace_bytes) + " of " +
                                       std::to_string(p.bytes) +
                                       " bytes or is not aligned to 256");
  DeviceScope scope;
  const int drc = scope.enter(device);
  if (drc != BSSCL_OK) return drc;
  (void)hipGetLastError();  // what an earlier call left is not this one's
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == BSSCL_BF16) return run_head<__bf16>(st, p, c);
  if (dtype == BSSCL_F16) return run_head<_Float16>(st, p, c);
  return run_head<float>(st, p, c);
}

}  // namespace

}  // namespace bsscl

using namespace bsscl;

extern "C" {

int bsscl_head_workspace(int32_t dtype, int64_t rows, int64_t width, int64_t vocab,
                         const void *weight, int64_t weight_stride, int32_t with_grad,
                         int64_t *bytes) {
  return no_throw([&] {
    if (!bytes) return set_error(BSSCL_EINVAL, "softmax head: null argument");
    HeadPlan p;
    const int rc = head_plan(dtype, rows, width, vocab, weight, weight_stride, with_grad != 0,
                             &p);
    if (rc == BSSCL_OK) *bytes = (int64_t)p.bytes;
    return rc;
  });
}

int bsscl_head_loss(int32_t device, void *stream, int32_t dtype, const void *hidden,
                    int64_t hidden_stride, const void *weight, int64_t weight_stride,
                    const int64_t *labels, const float *row_weight, int64_t rows, int64_t width,
                    int64_t vocab, int32_t reduction, double softcap, double z_loss, float *loss,
                    float *row_loss, float *lse, void *workspace, int64_t workspace_bytes) {
  return no_throw([&] {
    const HeadCall c{hidden, weight, hidden_stride, weight_stride, labels, row_weight,
                     reduction == BSSCL_MEAN, false, (float)softcap, (float)z_loss, 1.f, loss,
                     row_loss, lse, nullptr, nullptr, 0, 0, static_cast<char *>(workspace)};
    return head(device, stream, dtype, rows, width, vocab, reduction, workspace_bytes, c);
  });
}

int bsscl_head_grad(int32_t device, void *stream, int32_t dtype, const void *hidden,
                    int64_t hidden_stride, const void *weight, int64_t weight_stride,
                    const int64_t *labels, const float *row_weight, int64_t rows, int64_t width,
                    int64_t vocab, int32_t reduction, double softcap, double z_loss,
                    double grad_scale, float *loss, float *row_loss, float *lse, void *d_hidden,
                    int64_t d_hidden_stride, void *d_weight, int64_t d_weight_stride,
                    void *workspace, int64_t workspace_bytes) {
  return no_throw([&] {
    const HeadCall c{hidden, weight, hidden_stride, weight_stride, labels, row_weight,
                     reduction == BSSCL_MEAN, true, (float)softcap, (float)z_loss,
                     (float)grad_scale, loss, row_loss, lse, d_hidden, d_weight, d_hidden_stride,
                     d_weight_stride, static_cast<char *>(workspace)};
    return head(device, stream, dtype, rows, width, vocab, reduction, workspace_bytes, c);
  });
}

}  // extern "C"
