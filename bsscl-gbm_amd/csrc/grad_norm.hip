// The 2-norm over the values of many tensors, and the tensors scaled to it
// (the formulas stand in bsscl_hip.h).
//
// Bound by memory: the squares read everything once, the scaling reads it
// again and writes it.  The tensors' addresses and lengths travel as kernel
// arguments, up to kMostNorm (kMostClip) a launch, so nothing is copied to the
// device first and a captured launch keeps its list.  A launch's blocks take
// chunks of kChunk values in turn; a block keeps its sum of squares in float64
// (bf16 and float32 squares leave float32's range, and sums of billions lose
// float32's digits; the conversions and float64 products fill a third of the
// vector units at the memory's rate) and leaves it in a place of its own.
// Whoever needs the norm adds these, at most kBlocks a launch, in one fixed
// order: one block for the norm alone, each scaling block for itself, which
// saves clip_grads a launch.  The scaling takes the chunks in the opposite
// order, the last ones read first, while the last-level cache holds them.
// 1.9G bf16 values: squares 0.62 ms (6.0 TB/s), scaling 1.4 ms (5.4 TB/s);
// 157M values: 80 and 98 us.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <vector>

#include "device_call.h"
#include "wave.h"

namespace bsscl {

namespace {

constexpr int kMostNorm = 240, kMostClip = 160;  // tensors of a launch
constexpr int kChunk = 16384;                    // values a block takes at a time
constexpr int kBlocks = 2048;                    // of a launch, at most
constexpr int kThreads = 256;

// Tensors of a launch; bits 62 and 63 of a length hold the dtype.
struct NormList {
  const void *from[kMostNorm];
  uint64_t length[kMostNorm];
  int32_t count;
};
struct ClipList {
  const void *from[kMostClip];
  uint64_t length[kMostClip];
  int32_t count;
  void *to[kMostClip];
};
static_assert(sizeof(NormList) <= 4000 && sizeof(ClipList) <= 4000, "lists fit kernel arguments");
constexpr uint64_t kLengthMask = (uint64_t(1) << 62) - 1;

// Values before the first 16-byte boundary at or below p: chunks and vectors
// are counted from that boundary.
__host__ __device__ __forceinline__ uint32_t lead_of(const void *p, int dtype) {
  return (uint32_t)((uintptr_t)p & 15) / (dtype == BSSCL_F32 ? 4 : 2);
}

// first[t]: the first chunk of tensor t, first[count]: all of them.
template <typename L>
__device__ __forceinline__ void chunk_starts(const L &list, uint32_t *first, uint32_t *tmp) {
  const int t = (int)threadIdx.x;
  uint32_t n = 0;
  if (t < list.count) {
    const uint64_t len = list.length[t];
    n = (uint32_t)(((len & kLengthMask) + lead_of(list.from[t], (int)(len >> 62)) + kChunk - 1) /
                   kChunk);
  }
  const uint32_t incl = wave_incl_scan<uint32_t>(n);
  if ((t & 63) == 63) tmp[t >> 6] = incl;
  __syncthreads();
  uint32_t before = 0;
  for (int w = 0; w < (t >> 6); ++w) before += tmp[w];
  first[t + 1] = before + incl;
  if (t == 0) first[0] = 0;
  __syncthreads();
}

// Chunk c's tensor and its values [a, b), counted from the tensor's boundary.
struct ChunkAt {
  int t, dtype;
  int64_t a, b;
  uint32_t lead;
};
template <typename L>
__device__ __forceinline__ ChunkAt chunk_at(const L &list, const uint32_t *first, uint32_t c) {
  int lo = 0, hi = list.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (first[mid] <= c) lo = mid; else hi = mid - 1;
  }
  ChunkAt at;
  at.t = __builtin_amdgcn_readfirstlane(lo);
  const uint64_t len = list.length[at.t];
  at.dtype = (int)(len >> 62);
  at.lead = lead_of(list.from[at.t], at.dtype);
  at.a = (int64_t)(c - first[at.t]) * kChunk;
  const int64_t end = (int64_t)(len & kLengthMask) + at.lead;
  at.b = at.a + kChunk < end ? at.a + kChunk : end;
  return at;
}

template <typename F>
__device__ __forceinline__ void by_dtype(int dtype, F &&f) {
  if (dtype == BSSCL_BF16) f((__bf16 *)nullptr);
  else if (dtype == BSSCL_F16) f((_Float16 *)nullptr);
  else f((float *)nullptr);
}

template <typename T>
using Vec = T __attribute__((ext_vector_type(16 / sizeof(T))));

__device__ double block_sum(double v, double *tmp) {
  tmp[threadIdx.x] = v;
  for (int k = kThreads / 2; k > 0; k >>= 1) {
    __syncthreads();
    if ((int)threadIdx.x < k) tmp[threadIdx.x] += tmp[threadIdx.x + k];
  }
  __syncthreads();
  return tmp[0];
}

__global__ __launch_bounds__(kThreads) void k_squares(const NormList list, double *sums) {
  __shared__ uint32_t first[kThreads + 1], tmp4[4];
  __shared__ double tmp[kThreads];
  chunk_starts(list, first, tmp4);
  const uint32_t chunks = first[list.count];
  double s = 0.0;
  for (uint32_t c = blockIdx.x; c < chunks; c += gridDim.x) {
    const ChunkAt at = chunk_at(list, first, c);
    by_dtype(at.dtype, [&](auto *p) {
      using T = std::remove_pointer_t<decltype(p)>;
      constexpr int N = 16 / (int)sizeof(T), kBatch = 8;
      const T *x = static_cast<const T *>(list.from[at.t]) - at.lead;
      auto add = [&](T v) {
        const double d = (double)(float)v;
        s = fma(d, d, s);
      };
      const int64_t lead = at.a == 0 ? at.lead : at.a;  // the chunk's first value
      const int64_t a = (lead + N - 1) / N * N, b = at.b / N * N;
      if (a >= b) {
        for (int64_t i = lead + (int)threadIdx.x; i < at.b; i += kThreads) add(x[i]);
        return;
      }
      if ((int64_t)threadIdx.x < a - lead) add(x[lead + (int)threadIdx.x]);
      if ((int64_t)threadIdx.x < at.b - b) add(x[b + (int)threadIdx.x]);
      const Vec<T> *v = reinterpret_cast<const Vec<T> *>(x + a);
      const int n = (int)((b - a) / N);
      int i = (int)threadIdx.x;
      for (; i + (kBatch - 1) * kThreads < n; i += kBatch * kThreads) {
        Vec<T> y[kBatch];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) y[k] = v[i + k * kThreads];
#pragma unroll
        for (int k = 0; k < kBatch; ++k)
#pragma unroll
          for (int e = 0; e < N; ++e) add(y[k][e]);
      }
      for (; i < n; i += kThreads) {
        const Vec<T> y = v[i];
#pragma unroll
        for (int e = 0; e < N; ++e) add(y[e]);
      }
    });
  }
  s = block_sum(s, tmp);
  if (threadIdx.x == 0) sums[blockIdx.x] = s;
}

// |inv_scale| sqrt(sum of the launches' sums), the same in every block.
__device__ __forceinline__ double norm_of(const double *sums, int32_t count, double inv_scale,
                                          double *tmp) {
  double s = 0.0;
  int32_t i = (int)threadIdx.x;
  for (; i + 7 * kThreads < count; i += 8 * kThreads) {
    double y[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) y[k] = sums[i + k * kThreads];
#pragma unroll
    for (int k = 0; k < 8; ++k) s += y[k];
  }
  for (; i < count; i += kThreads) s += sums[i];
  return fabs(inv_scale) * sqrt(block_sum(s, tmp));
}

__global__ __launch_bounds__(kThreads) void k_norm(const double *sums, int32_t count,
                                                   double inv_scale, float *norm_out) {
  __shared__ double tmp[kThreads];
  const double norm = norm_of(sums, count, inv_scale, tmp);
  if (threadIdx.x == 0) *norm_out = (float)norm;
}

__global__ __launch_bounds__(kThreads) void k_scale(const ClipList list, const double *sums,
                                                    int32_t count, double inv_scale,
                                                    double max_norm, float *norm_out) {
  __shared__ uint32_t first[kThreads + 1], tmp4[4];
  __shared__ double tmp[kThreads];
  const double norm = norm_of(sums, count, inv_scale, tmp);
  if (blockIdx.x == 0 && threadIdx.x == 0 && norm_out) *norm_out = (float)norm;
  const double f =
      norm > max_norm && (float)norm < INFINITY ? inv_scale * (max_norm / norm) : inv_scale;
  // Below float32's normal range the factor is kept as fa times a power of
  // two, so that no digits of it are lost.
  const bool small = fabs(f) < 0x1p-126;
  const float fa = (float)(small ? f * 0x1p126 : f), fb = small ? 0x1p-126f : 1.f;
  chunk_starts(list, first, tmp4);
  const uint32_t chunks = first[list.count];
  for (uint32_t c = blockIdx.x; c < chunks; c += gridDim.x) {
    const ChunkAt at = chunk_at(list, first, chunks - 1 - c);
    by_dtype(at.dtype, [&](auto *p) {
      using T = std::remove_pointer_t<decltype(p)>;
      constexpr int N = 16 / (int)sizeof(T), kBatch = 8;
      const T *x = static_cast<const T *>(list.from[at.t]);
      T *o = static_cast<T *>(list.to[at.t]);
      if (fa == 1.f && !small && x == o) return;
      const bool whole = (((uintptr_t)x ^ (uintptr_t)o) & 15) == 0;
      x -= at.lead;
      o -= at.lead;
      auto put = [&](int64_t i) { o[i] = (T)((float)x[i] * fa * fb); };
      const int64_t lead = at.a == 0 ? at.lead : at.a;
      const int64_t a = (lead + N - 1) / N * N, b = at.b / N * N;
      if (a >= b || !whole) {
        for (int64_t i = lead + (int)threadIdx.x; i < at.b; i += kThreads) put(i);
        return;
      }
      if ((int64_t)threadIdx.x < a - lead) put(lead + (int)threadIdx.x);
      if ((int64_t)threadIdx.x < at.b - b) put(b + (int)threadIdx.x);
      const Vec<T> *v = reinterpret_cast<const Vec<T> *>(x + a);
      Vec<T> *w = reinterpret_cast<Vec<T> *>(o + a);
      const int n = (int)((b - a) / N);
      auto scaled = [&](Vec<T> y) {
#pragma unroll
        for (int e = 0; e < N; ++e) y[e] = (T)((float)y[e] * fa * fb);
        return y;
      };
      int i = (int)threadIdx.x;
      for (; i + (kBatch - 1) * kThreads < n; i += kBatch * kThreads) {
        Vec<T> y[kBatch];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) y[k] = v[i + k * kThreads];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) w[i + k * kThreads] = scaled(y[k]);
      }
      for (; i < n; i += kThreads) w[i] = scaled(v[i]);
    });
  }
}

// Chunks of the tensors that launches of `most` take together, at most:
// a tensor off a 16-byte boundary may touch one more than its length says.
int sums_of(int32_t count, const int64_t *lengths, int64_t *sums) {
  if (count < 0 || (count > 0 && !lengths))
    return set_error(BSSCL_EINVAL, "gradient norm: null or negative list");
  int64_t chunks = 0;
  for (int32_t t = 0; t < count; ++t) {
    if (lengths[t] < 0 || lengths[t] > (int64_t(1) << 40))
      return set_error(BSSCL_EINVAL, "gradient norm: a length must be in [0, 2^40]");
    if (lengths[t]) chunks += lengths[t] / kChunk + 2;
  }
  if (chunks >= (int64_t(1) << 31))
    return set_error(BSSCL_EINVAL, "gradient norm: too many values");
  *sums = std::max<int64_t>(
      32, std::min<int64_t>(chunks, ((int64_t)count / kMostClip + 1) * kBlocks));
  return BSSCL_OK;
}

int check_list(int32_t count, const void *const *tensors, void *const *out, const int64_t *lengths,
               const int32_t *dtypes) {
  if (count > 0 && (!tensors || !dtypes))
    return set_error(BSSCL_EINVAL, "gradient norm: null list");
  struct Range {
    uintptr_t a, b;
    int32_t t;
    bool out;
  };
  std::vector<Range> ranges;
  for (int32_t t = 0; t < count; ++t) {
    if (dtypes[t] != BSSCL_BF16 && dtypes[t] != BSSCL_F16 && dtypes[t] != BSSCL_F32)
      return set_error(BSSCL_EINVAL, "gradient norm: unknown dtype " + std::to_string(dtypes[t]));
    if (lengths[t] == 0) continue;
    const uintptr_t size = dtypes[t] == BSSCL_F32 ? 4 : 2;
    const uintptr_t a = (uintptr_t)tensors[t], bytes = (uintptr_t)lengths[t] * size;
    if (!a || a % size) return set_error(BSSCL_EINVAL, "gradient norm: null or misaligned tensor");
    if (!out) continue;
    const uintptr_t o = (uintptr_t)out[t];
    if (!o || o % size) return set_error(BSSCL_EINVAL, "clip_grads: null or misaligned out");
    ranges.push_back({o, o + bytes, t, true});
    if (o != a) ranges.push_back({a, a + bytes, t, false});
  }
  // Sorted by address, a range that begins before an out range ends (or an
  // out range that begins before any range ends) overlaps it.
  std::sort(ranges.begin(), ranges.end(), [](const Range &x, const Range &y) { return x.a < y.a; });
  uintptr_t end_out = 0, end_any = 0;
  for (const Range &r : ranges) {
    if (r.a < end_out || (r.out && r.a < end_any))
      return set_error(BSSCL_EINVAL, "clip_grads: the out of tensor " + std::to_string(r.t) +
                                         " or one beside it overlaps another tensor");
    end_any = std::max(end_any, r.b);
    if (r.out) end_out = std::max(end_out, r.b);
  }
  return BSSCL_OK;
}

// f(list, its blocks) for each launch's part of the tensors.
template <typename L, int MOST, typename F>
int for_launches(int32_t count, const void *const *tensors, void *const *out,
                 const int64_t *lengths, const int32_t *dtypes, F &&f) {
  L list;
  for (int32_t t = 0; t < count;) {
    list.count = 0;
    int64_t chunks = 0;
    for (; t < count && list.count < MOST; ++t) {
      if (lengths[t] == 0) continue;
      const int k = list.count++;
      list.from[k] = tensors[t];
      list.length[k] = (uint64_t)lengths[t] | (uint64_t)dtypes[t] << 62;
      if constexpr (std::is_same<L, ClipList>::value) list.to[k] = out[t];
      chunks += (lengths[t] + lead_of(tensors[t], dtypes[t]) + kChunk - 1) / kChunk;
    }
    if (list.count) f(list, (unsigned)std::min<int64_t>(chunks, kBlocks));
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess)
    return set_error(BSSCL_EDEVICE, std::string("gradient norm: ") + hipGetErrorString(e));
  return BSSCL_OK;
}

int norm_and_clip(int32_t device, void *stream, int32_t count, const void *const *tensors,
                  void *const *out, const int64_t *lengths, const int32_t *dtypes,
                  double inv_scale, double max_norm, float *norm, void *workspace,
                  int64_t workspace_bytes) {
  int64_t most = 0;
  int rc = sums_of(count, lengths, &most);
  if (rc == BSSCL_OK) rc = check_list(count, tensors, out, lengths, dtypes);
  if (rc != BSSCL_OK) return rc;
  if (!std::isfinite((float)inv_scale))  // (an infinite factor would make zeros NaN)
    return set_error(BSSCL_EINVAL, "gradient norm: inv_scale must be finite in float32");
  if (!norm || !workspace || ((uintptr_t)workspace & 255) ||
      workspace_bytes < most * (int64_t)sizeof(double))
    return set_error(BSSCL_EINVAL,
                     "gradient norm: null norm, or a null, short or unaligned workspace");
  DeviceScope scope;
  rc = scope.enter(device);
  if (rc != BSSCL_OK) return rc;
  (void)hipGetLastError();  // what an earlier call left is not this one's
  hipStream_t st = static_cast<hipStream_t>(stream);
  auto *sums = static_cast<double *>(workspace);
  int32_t n = 0;
  rc = for_launches<NormList, kMostNorm>(count, tensors, nullptr, lengths, dtypes,
                                         [&](const NormList &list, unsigned blocks) {
                                           k_squares<<<blocks, kThreads, 0, st>>>(list, sums + n);
                                           n += (int32_t)blocks;
                                         });
  if (rc != BSSCL_OK) return rc;
  bool told = false;
  if (out)
    rc = for_launches<ClipList, kMostClip>(
        count, tensors, out, lengths, dtypes, [&](const ClipList &list, unsigned blocks) {
          k_scale<<<blocks, kThreads, 0, st>>>(list, sums, n, inv_scale, max_norm,
                                               told ? nullptr : norm);
          told = true;
        });
  if (rc == BSSCL_OK && !told) {
    k_norm<<<1, kThreads, 0, st>>>(sums, n, inv_scale, norm);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess)
      return set_error(BSSCL_EDEVICE, std::string("gradient norm: ") + hipGetErrorString(e));
  }
  return rc;
}

}  // namespace

}  // namespace bsscl

using namespace bsscl;

extern "C" {

int bsscl_grad_norm_workspace(int32_t count, const int64_t *lengths, int64_t *bytes) {
  return no_throw([&] {
    int64_t sums = 0;
    if (!bytes) return set_error(BSSCL_EINVAL, "gradient norm: null argument");
    const int rc = sums_of(count, lengths, &sums);
    if (rc == BSSCL_OK) *bytes = sums * (int64_t)sizeof(double);
    return rc;
  });
}

int bsscl_grad_norm(int32_t device, void *stream, int32_t count, const void *const *tensors,
                    const int64_t *lengths, const int32_t *dtypes, double inv_scale, float *norm,
                    void *workspace, int64_t workspace_bytes) {
  return no_throw([&] {
    return norm_and_clip(device, stream, count, tensors, nullptr, lengths, dtypes, inv_scale, 0.0,
                         norm, workspace, workspace_bytes);
  });
}

int bsscl_clip_grads(int32_t device, void *stream, int32_t count, const void *const *tensors,
                     void *const *out, const int64_t *lengths, const int32_t *dtypes,
                     double inv_scale, double max_norm, float *norm, void *workspace,
                     int64_t workspace_bytes) {
  return no_throw([&] {
    if (count > 0 && !out) return set_error(BSSCL_EINVAL, "clip_grads: null out");
    if (!(max_norm >= 0.0)) return set_error(BSSCL_EINVAL, "clip_grads: max_norm must be >= 0");
    return norm_and_clip(device, stream, count, tensors, out, lengths, dtypes, inv_scale, max_norm,
                         norm, workspace, workspace_bytes);
  });
}

}  // extern "C"
