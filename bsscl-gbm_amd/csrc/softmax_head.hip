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
// row and tile, exp(m_t - lse) times the row's weight, and puts the label's
// own value there from its float32 score, where p - 1 keeps what a rounded p
// would lose.  These rows of the vocabulary's length are made for a piece of
// the rows at a time (kPieceBytes), and both products consume a piece before
// the next one takes its place.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "device_call.h"

namespace bsscl {

namespace {

constexpr int kTileV = 64;      // classes of a score tile
constexpr int kTileR = 64;      // rows of a score tile
constexpr int kRowPad = 256;    // rows of a piece: a multiple
constexpr int kColPad = 64;     // width of the packed rows: a multiple
constexpr int64_t kPieceBytes = int64_t(1) << 30;

struct HeadInfo {
  int32_t rows;      // counting rows
  float to_operand;  // power of two on d loss / d score in the operands (float16)
  float from_operand;
};

// A tile's exponentials, at most 1, are kept times this: in float16 they would
// lose digits below 2^-14 of the tile's maximum otherwise.
template <typename T>
constexpr float kExpScale = std::is_same<T, _Float16>::value ? 32768.f : 1.f;

template <typename T>
__device__ __forceinline__ T from_float(float x) {
  if constexpr (std::is_same<T, _Float16>::value)
    x = fminf(fmaxf(x, -65504.f), 65504.f);
  return (T)x;
}

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

// Sum over the block's 1024 threads in a fixed order, in every thread.
__device__ double block_sum_1024(double v, double *tmp) {
  __syncthreads();
  tmp[threadIdx.x] = v;
  for (int k = 512; k > 0; k >>= 1) {
    __syncthreads();
    if ((int)threadIdx.x < k) tmp[threadIdx.x] += tmp[threadIdx.x + k];
  }
  __syncthreads();
  return tmp[0];
}

// One block: the counting rows in order (idx, their labels and final weights),
// the place of each row (pos, -1 for none) and the zeros of the rows left out.
__global__ __launch_bounds__(1024) void k_head_prepare(
    const int64_t *labels, const float *row_weight, int32_t rows, int32_t vocab, int32_t mean,
    float grad_scale, int32_t narrow, int32_t *idx, int32_t *lab, float *u, int32_t *pos,
    float *row_loss, float *lse, HeadInfo *info) {
  __shared__ int32_t wave_count[16];
  __shared__ double tmp[1024];
  __shared__ float top[1024];
  const int tid = (int)threadIdx.x, lane = tid & 63, wid = tid >> 6;
  int32_t base = 0;
  double sum = 0.0;
  float big = 0.f;
  for (int32_t at = 0; at < rows; at += 1024) {
    const int32_t i = at + tid;
    const int64_t y = i < rows ? labels[i] : -1;
    const bool counts = y >= 0 && y < vocab;
    const unsigned long long mask = __ballot(counts);
    if (lane == 0) wave_count[wid] = __popcll(mask);
    __syncthreads();
    int32_t before = base, all = 0;
    for (int w = 0; w < 16; ++w) {
      const int32_t c = wave_count[w];
      before += w < wid ? c : 0;
      all += c;
    }
    base += all;
    __syncthreads();
    if (i >= rows) continue;
    const int32_t p = before + __popcll(mask & ((1ull << lane) - 1));
    pos[i] = counts ? p : -1;
    if (counts) {
      const float w = row_weight ? row_weight[i] : 1.f;
      idx[p] = i;
      lab[p] = (int32_t)y;
      u[p] = w;
      sum += (double)w;
      big = fmaxf(big, fabsf(w));
    } else {
      row_loss[i] = 0.f;
      lse[i] = 0.f;
    }
  }
  sum = block_sum_1024(sum, tmp);
  top[tid] = big;
  for (int k = 512; k > 0; k >>= 1) {
    __syncthreads();
    if (tid < k) top[tid] = fmaxf(top[tid], top[tid + k]);
  }
  __syncthreads();
  const double share = mean ? (sum != 0.0 ? 1.0 / sum : 0.0) : 1.0;
  if (tid == 0) {
    // The largest weight at 2^10 to 2^11 leaves a factor of 2^5 to float16's largest
    // value (1 + 2 zeta lse may exceed 1) and its smallest at 2^-35 of the weight.
    int e = 0;
    const float m = (float)(top[0] * fabs(share)) * fabsf(grad_scale);
    if (narrow && m > 0.f && m < INFINITY) e = 10 - ilogbf(m);
    e = e < -100 ? -100 : e > 100 ? 100 : e;
    info->rows = base;
    info->to_operand = ldexpf(1.f, e);
    info->from_operand = ldexpf(1.f, -e);
  }
  if (mean)
    for (int32_t p = tid; p < base; p += 1024) u[p] = (float)((double)u[p] * share);
}

// Block b < rows: row b to its place among the counting rows, widened with
// zeros to `wide`, or zeros into d_hidden.  The blocks after them: zero rows
// up to the next multiple of kRowPad.
template <typename T>
__global__ __launch_bounds__(256) void k_pack_hidden(const T *hidden, int64_t stride, int32_t rows,
                                                     int32_t width, int32_t wide,
                                                     const int32_t *pos, const HeadInfo *info,
                                                     T *packed, T *d_hidden, int64_t d_stride) {
  const int32_t b = (int32_t)blockIdx.x;
  if (b >= rows) {
    const int32_t n = info->rows, p = n + (b - rows);
    if (p >= (n + kRowPad - 1) / kRowPad * kRowPad) return;
    for (int32_t d = (int32_t)threadIdx.x; d < wide; d += 256) packed[(int64_t)p * wide + d] = (T)0.f;
    return;
  }
  const int32_t p = pos[b];
  if (p >= 0) {
    const T *from = hidden + (int64_t)b * stride;
    for (int32_t d = (int32_t)threadIdx.x; d < wide; d += 256)
      packed[(int64_t)p * wide + d] = d < width ? from[d] : (T)0.f;
  } else if (d_hidden) {
    for (int32_t d = (int32_t)threadIdx.x; d < width; d += 256)
      d_hidden[(int64_t)b * d_stride + d] = (T)0.f;
  }
}

// 64 x 64 tile of sum_k A(m, k) B(n, k) in float32: thread (tx, ty) of 16 x 16
// holds m = 4 ty + 0..3, n = 4 tx + 0..3.  A and B give 0 outside.
template <typename FA, typename FB>
__device__ void mm_tile(FA A, FB B, int64_t k_end, float (&acc)[4][4]) {
  __shared__ float sa[16][65], sb[16][65];
  const int tx = (int)threadIdx.x & 15, ty = (int)threadIdx.x >> 4;
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) acc[i][j] = 0.f;
  for (int64_t k0 = 0; k0 < k_end; k0 += 16) {
    for (int e = (int)threadIdx.x; e < 1024; e += 256) {
      sa[e & 15][e >> 4] = A(e >> 4, k0 + (e & 15));
      sb[e & 15][e >> 4] = B(e >> 4, k0 + (e & 15));
    }
    __syncthreads();
    for (int k = 0; k < 16; ++k)
      for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) acc[i][j] += sa[k][4 * ty + i] * sb[k][4 * tx + j];
    __syncthreads();
  }
}

// One score tile: kTileV classes x kTileR rows.
template <typename T>
__global__ __launch_bounds__(256) void k_scores(const T *weight, int64_t w_stride, int32_t vocab,
                                                int32_t width, const T *packed, int32_t wide,
                                                const int32_t *lab, const HeadInfo *info,
                                                int32_t piece, int32_t pieces, float softcap,
                                                int32_t tiles, float2 *stats, float *z_label, T *P,
                                                int64_t ldp) {
  __shared__ float z[kTileR][kTileV + 1];
  const Piece pc = piece_of(info->rows, piece, pieces);
  const int32_t r0 = (int32_t)blockIdx.y * kTileR, v0 = (int32_t)blockIdx.x * kTileV;
  if (r0 >= pc.rows) return;
  const T *h = packed + ((int64_t)pc.begin + r0) * wide;
  float acc[4][4];
  mm_tile(
      [&](int m, int64_t k) {
        return v0 + m < vocab && k < width ? (float)weight[(int64_t)(v0 + m) * w_stride + k] : 0.f;
      },
      [&](int n, int64_t k) { return k < wide ? (float)h[(int64_t)n * wide + k] : 0.f; }, width, acc);
  const int tx = (int)threadIdx.x & 15, ty = (int)threadIdx.x >> 4;
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      float s = acc[i][j];
      if (softcap > 0.f) s = softcap * tanhf(s / softcap);
      z[4 * tx + j][4 * ty + i] = v0 + 4 * ty + i < vocab ? s : -INFINITY;
    }
  __syncthreads();
  const int n = (int)threadIdx.x;
  if (n < kTileR) {
    const int32_t r = r0 + n;
    float m = -INFINITY, s = 0.f;
    for (int v = 0; v < kTileV; ++v) m = fmaxf(m, z[n][v]);
    if (r < pc.rows) {
      const int32_t y = lab[pc.begin + r] - v0;
      if (y >= 0 && y < kTileV) z_label[r] = z[n][y];
    }
    const float base = m == -INFINITY ? 0.f : m;
    for (int v = 0; v < kTileV; ++v) {
      const float zv = z[n][v], e = expf(zv - base);
      s += e;
      const float slope = softcap > 0.f && e > 0.f ? 1.f - (zv / softcap) * (zv / softcap) : 1.f;
      z[n][v] = e * slope * kExpScale<T>;
    }
    if (r < pc.rows) stats[(int64_t)r * tiles + blockIdx.x] = make_float2(m, s);
  }
  if (!P) return;
  __syncthreads();
  for (int e = (int)threadIdx.x; e < kTileR * kTileV; e += 256)
    P[(int64_t)(r0 + (e >> 6)) * ldp + v0 + (e & 63)] = (T)z[e >> 6][e & 63];
}

// One block per row of the piece: lse and loss from the tiles' statistics;
// with P, the row of d loss / d score in its place.
template <typename T>
__global__ __launch_bounds__(256) void k_rows(const HeadInfo *info, int32_t piece, int32_t pieces,
                                              const int32_t *idx, const int32_t *lab,
                                              const float *u, float softcap, float z_loss,
                                              float grad_scale, int32_t tiles,
                                              const float2 *stats, const float *z_label, T *P,
                                              int64_t ldp, float *row_loss, float *lse_out) {
  __shared__ float red[256];
  const Piece pc = piece_of(info->rows, piece, pieces);
  const int32_t r = (int32_t)blockIdx.x;
  const int tid = (int)threadIdx.x;
  if (r >= pc.rows) {
    // The products read whole steps of rows: zeros behind the last one.
    if (P && r < (pc.rows + kRowPad - 1) / kRowPad * kRowPad)
      for (int64_t v = tid; v < ldp; v += 256) P[(int64_t)r * ldp + v] = (T)0.f;
    return;
  }
  const float2 *st = stats + (int64_t)r * tiles;
  float m = -INFINITY;
  for (int t = tid; t < tiles; t += 256) m = fmaxf(m, st[t].x);
  red[tid] = m;
  for (int k = 128; k > 0; k >>= 1) {
    __syncthreads();
    if (tid < k) red[tid] = fmaxf(red[tid], red[tid + k]);
  }
  __syncthreads();
  m = red[0];
  const float base = m == -INFINITY ? 0.f : m;
  float s = 0.f;
  for (int t = tid; t < tiles; t += 256) s += st[t].y * expf(st[t].x - base);
  __syncthreads();
  red[tid] = s;
  for (int k = 128; k > 0; k >>= 1) {
    __syncthreads();
    if (tid < k) red[tid] += red[tid + k];
  }
  __syncthreads();
  const float lse = base + logf(red[0]);
  const int32_t c = pc.begin + r, y = lab[c];
  const float zy = z_label[r];
  if (tid == 0) {
    row_loss[idx[c]] = lse - zy + z_loss * lse * lse;
    lse_out[idx[c]] = lse;
  }
  if (!P) return;
  const float g = u[c] * grad_scale * info->to_operand, zl = 2.f * z_loss * lse;
  const float py = expm1f(zy - lse);
  const float slope = softcap > 0.f ? 1.f - (zy / softcap) * (zy / softcap) : 1.f;
  const float own = g * slope * (py + zl * (py + 1.f));
  T *row = P + (int64_t)r * ldp;
  for (int64_t v = tid; v < ldp; v += 256) {
    const float f = expf(st[v / kTileV].x - lse) * (g * (1.f + zl) / kExpScale<T>);
    row[v] = from_float<T>(v == y ? own : (float)row[v] * f);
  }
}

// d_hidden of a piece: rows x width, over the whole vocabulary.
template <typename T>
__global__ __launch_bounds__(256) void k_d_hidden(const T *P, int64_t ldp, const T *weight,
                                                  int64_t w_stride, int32_t vocab, int32_t width,
                                                  const HeadInfo *info, int32_t piece,
                                                  int32_t pieces, const int32_t *idx, T *d_hidden,
                                                  int64_t d_stride) {
  const Piece pc = piece_of(info->rows, piece, pieces);
  const int32_t r0 = (int32_t)blockIdx.y * 64, d0 = (int32_t)blockIdx.x * 64;
  if (r0 >= pc.rows) return;
  float acc[4][4];
  mm_tile(
      [&](int m, int64_t k) {
        return d0 + m < width && k < vocab ? (float)weight[k * w_stride + d0 + m] : 0.f;
      },
      [&](int n, int64_t k) { return k < vocab ? (float)P[(int64_t)(r0 + n) * ldp + k] : 0.f; },
      vocab, acc);
  const int tx = (int)threadIdx.x & 15, ty = (int)threadIdx.x >> 4;
  for (int j = 0; j < 4; ++j) {
    const int32_t r = r0 + 4 * tx + j;
    if (r >= pc.rows) continue;
    T *out = d_hidden + (int64_t)idx[pc.begin + r] * d_stride;
    for (int i = 0; i < 4; ++i)
      if (d0 + 4 * ty + i < width) out[d0 + 4 * ty + i] = (T)(acc[i][j] * info->from_operand);
  }
}

// d_weight of a piece: vocab x width, over the piece's rows; pieces before the
// last add up in float32.
template <typename T>
__global__ __launch_bounds__(256) void k_d_weight(const T *P, int64_t ldp, const T *packed,
                                                  int32_t wide, int32_t vocab, int32_t width,
                                                  const HeadInfo *info, int32_t piece,
                                                  int32_t pieces, float *sum, T *d_weight,
                                                  int64_t d_stride) {
  const Piece pc = piece_of(info->rows, piece, pieces);
  const int32_t v0 = (int32_t)blockIdx.y * 64, d0 = (int32_t)blockIdx.x * 64;
  const T *h = packed + (int64_t)pc.begin * wide;
  float acc[4][4];
  mm_tile(
      [&](int m, int64_t k) {
        return d0 + m < wide && k < pc.rows ? (float)h[k * wide + d0 + m] : 0.f;
      },
      [&](int n, int64_t k) { return k < pc.rows ? (float)P[k * ldp + v0 + n] : 0.f; }, pc.rows,
      acc);
  const int tx = (int)threadIdx.x & 15, ty = (int)threadIdx.x >> 4;
  for (int j = 0; j < 4; ++j) {
    const int32_t v = v0 + 4 * tx + j;
    if (v >= vocab) continue;
    for (int i = 0; i < 4; ++i) {
      const int32_t d = d0 + 4 * ty + i;
      if (d >= width) continue;
      float x = acc[i][j];
      if (piece > 0) x += sum[(int64_t)v * wide + d];
      if (piece < pieces - 1)
        sum[(int64_t)v * wide + d] = x;
      else
        d_weight[(int64_t)v * d_stride + d] = (T)(x * info->from_operand);
    }
  }
}

// loss = sum of u * row_loss over the counting rows, in their order.
__global__ __launch_bounds__(1024) void k_loss_sum(const HeadInfo *info, const int32_t *idx,
                                                   const float *u, const float *row_loss,
                                                   float *loss) {
  __shared__ double tmp[1024];
  double s = 0.0;
  for (int32_t p = (int32_t)threadIdx.x; p < info->rows; p += 1024)
    s += (double)u[p] * (double)row_loss[idx[p]];
  s = block_sum_1024(s, tmp);
  if (threadIdx.x == 0) *loss = (float)s;
}

// Where a call's intermediate values lie in its workspace.
struct HeadPlan {
  int32_t rows, width, wide, vocab, tiles;
  int32_t piece_rows, pieces;
  int64_t ldp;
  size_t info, idx, lab, u, pos, packed, stats, z_label, P, sum, bytes;
};

int head_plan(int32_t dtype, int64_t rows, int64_t width, int64_t vocab, bool grad, HeadPlan *pl) {
  if (dtype != BSSCL_BF16 && dtype != BSSCL_F16 && dtype != BSSCL_F32)
    return set_error(BSSCL_EINVAL, "softmax head: unknown dtype " + std::to_string(dtype));
  if (rows < 1 || vocab < 1 || width < 1 || rows >= (1 << 30) || vocab >= (1 << 30) ||
      width > 65536)
    return set_error(BSSCL_EINVAL,
                     "softmax head: rows and vocab must be in [1, 2^30), width in [1, 65536]");
  const int64_t es = dtype == BSSCL_F32 ? 4 : 2;
  HeadPlan p{};
  p.rows = (int32_t)rows;
  p.width = (int32_t)width;
  p.wide = (int32_t)round_up(width, kColPad);
  p.vocab = (int32_t)vocab;
  p.tiles = (int32_t)((vocab + kTileV - 1) / kTileV);
  p.ldp = (int64_t)p.tiles * kTileV;
  const int64_t row_bytes = grad ? p.ldp * es : (int64_t)p.tiles * (int64_t)sizeof(float2);
  const int64_t fit = std::max<int64_t>(kRowPad, kPieceBytes / row_bytes / kRowPad * kRowPad);
  p.piece_rows = (int32_t)std::min<int64_t>(fit, round_up(rows, kRowPad));
  p.pieces = (int32_t)((rows + p.piece_rows - 1) / p.piece_rows);
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
  p.P = take(grad ? (int64_t)p.piece_rows * p.ldp * es : 0);
  p.sum = take(grad && p.pieces > 1 ? vocab * p.wide * 4 : 0);
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
  auto *P = c.grad ? reinterpret_cast<T *>(c.ws + p.P) : nullptr;
  auto *sum = reinterpret_cast<float *>(c.ws + p.sum);
  auto *weight = static_cast<const T *>(c.weight);
  k_head_prepare<<<1, 1024, 0, st>>>(c.labels, c.row_weight, p.rows, p.vocab, c.mean,
                                     c.grad_scale, std::is_same<T, _Float16>::value, idx, lab, u,
                                     pos, c.row_loss, c.lse, info);
  k_pack_hidden<T><<<p.rows + kRowPad, 256, 0, st>>>(
      static_cast<const T *>(c.hidden), c.h_stride, p.rows, p.width, p.wide, pos, info, packed,
      static_cast<T *>(c.d_hidden), c.dh_stride);
  for (int32_t k = 0; k < p.pieces; ++k) {
    const unsigned row_tiles = (unsigned)(p.piece_rows / kTileR);
    k_scores<T><<<dim3((unsigned)p.tiles, row_tiles), 256, 0, st>>>(
        weight, c.w_stride, p.vocab, p.width, packed, p.wide, lab, info, k, p.pieces, c.softcap,
        p.tiles, stats, z_label, P, p.ldp);
    k_rows<T><<<p.piece_rows, 256, 0, st>>>(info, k, p.pieces, idx, lab, u, c.softcap, c.z_loss,
                                            c.grad_scale, p.tiles, stats, z_label, P, p.ldp,
                                            c.row_loss, c.lse);
    if (!c.grad) continue;
    const unsigned cols = (unsigned)((p.width + 63) / 64);
    k_d_hidden<T><<<dim3(cols, row_tiles), 256, 0, st>>>(P, p.ldp, weight, c.w_stride, p.vocab,
                                                         p.width, info, k, p.pieces, idx,
                                                         static_cast<T *>(c.d_hidden), c.dh_stride);
    k_d_weight<T><<<dim3(cols, (unsigned)p.tiles), 256, 0, st>>>(
        P, p.ldp, packed, p.wide, p.vocab, p.width, info, k, p.pieces, sum,
        static_cast<T *>(c.d_weight), c.dw_stride);
  }
  k_loss_sum<<<1, 1024, 0, st>>>(info, idx, u, c.row_loss, c.loss);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess)
    return set_error(BSSCL_EDEVICE, std::string("softmax head: ") + hipGetErrorString(e));
  return BSSCL_OK;
}

int head(int32_t device, void *stream, int32_t dtype, int64_t rows, int64_t width, int64_t vocab,
         int32_t reduction, int64_t workspace_bytes, const HeadCall &c) {
  HeadPlan p;
  const int rc = head_plan(dtype, rows, width, vocab, c.grad, &p);
  if (rc != BSSCL_OK) return rc;
  if (!c.hidden || !c.weight || !c.labels || !c.loss || !c.row_loss || !c.lse || !c.ws ||
      (c.grad && (!c.d_hidden || !c.d_weight)))
    return set_error(BSSCL_EINVAL, "softmax head: null argument");
  if (c.h_stride < width || c.w_stride < width ||
      (c.grad && (c.dh_stride < width || c.dw_stride < width)))
    return set_error(BSSCL_EINVAL, "softmax head: a row stride is below the width");
  if (reduction != BSSCL_SUM && reduction != BSSCL_MEAN)
    return set_error(BSSCL_EINVAL, "softmax head: unknown reduction");
  if (!(c.softcap >= 0.f) || !std::isfinite(c.softcap) || !(c.z_loss >= 0.f) ||
      !std::isfinite(c.z_loss) || !std::isfinite(c.grad_scale))
    return set_error(BSSCL_EINVAL,
                     "softmax head: softcap and z_loss must be finite and >= 0, grad_scale finite");
  if ((size_t)workspace_bytes < p.bytes || ((uintptr_t)c.ws & 255))
    return set_error(BSSCL_EINVAL, "softmax head: the workspace holds " +
                                       std::to_string(workspace_bytes) + " of " +
                                       std::to_string(p.bytes) +
                                       " bytes or is not aligned to 256");
  DeviceScope scope;
  const int drc = scope.enter(device);
  if (drc != BSSCL_OK) return drc;
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
    const int rc = head_plan(dtype, rows, width, vocab, with_grad != 0, &p);
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
