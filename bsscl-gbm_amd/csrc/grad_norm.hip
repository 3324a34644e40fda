// The 2-norm over the values of many tensors, and the tensors scaled to it
// (the formulas stand in bsscl_hip.h).
//
// The tensors' addresses and lengths travel as kernel arguments, up to
// kPerLaunch tensors a launch, so nothing is copied to the device first and a
// captured launch keeps its list.  A block's values come from one chunk of one
// tensor; its sum of squares in float64 (bf16 and float32 squares leave
// float32's range, and sums of billions lose float32's digits) goes to a place
// of its own, and one block adds these in a fixed order.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <vector>

#include "device_call.h"

namespace bsscl {

namespace {

constexpr int kPerLaunch = 112;
constexpr int kChunk = 16384;  // values of a block
constexpr int64_t kMaxBlocks = int64_t(1) << 31;

struct TensorList {
  const void *from[kPerLaunch];
  void *to[kPerLaunch];
  int64_t length[kPerLaunch];
  uint32_t first[kPerLaunch + 1];  // first block of each tensor in this launch
  uint8_t dtype[kPerLaunch];
  int32_t count;
};
static_assert(sizeof(TensorList) <= 3500, "the list fits the kernel arguments");

// The factor is a * b: below float32's normal range b is a power of two that
// keeps the digits of a.
struct NormInfo {
  float a, b;
};

// The tensor of block b: the last one whose first block is not above b.
__device__ __forceinline__ int tensor_of(const TensorList &L, uint32_t b) {
  int lo = 0, hi = L.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (L.first[mid] <= b) lo = mid; else hi = mid - 1;
  }
  return lo;
}

template <typename F>
__device__ __forceinline__ void by_dtype(int dtype, F &&f) {
  if (dtype == BSSCL_BF16) f((__bf16 *)nullptr);
  else if (dtype == BSSCL_F16) f((_Float16 *)nullptr);
  else f((float *)nullptr);
}

__device__ double block_sum_256(double v, double *tmp) {
  tmp[threadIdx.x] = v;
  for (int k = 128; k > 0; k >>= 1) {
    __syncthreads();
    if ((int)threadIdx.x < k) tmp[threadIdx.x] += tmp[threadIdx.x + k];
  }
  __syncthreads();
  return tmp[0];
}

__global__ __launch_bounds__(256) void k_squares(const TensorList L, double *sums) {
  __shared__ double tmp[256];
  const int t = tensor_of(L, blockIdx.x);
  const int64_t a = (int64_t)(blockIdx.x - L.first[t]) * kChunk;
  const int64_t b = a + kChunk < L.length[t] ? a + kChunk : L.length[t];
  double s = 0.0;
  by_dtype(L.dtype[t], [&](auto *p) {
    auto *x = static_cast<decltype(p)>(const_cast<void *>(L.from[t]));
    for (int64_t i = a + (int)threadIdx.x; i < b; i += 256) {
      const double v = (double)(float)x[i];
      s += v * v;
    }
  });
  s = block_sum_256(s, tmp);
  if (threadIdx.x == 0) sums[blockIdx.x] = s;
}

__global__ __launch_bounds__(256) void k_norm(const double *sums, int64_t blocks, double inv_scale,
                                              double max_norm, float *norm_out, NormInfo *info) {
  __shared__ double tmp[256];
  double s = 0.0;
  for (int64_t i = (int)threadIdx.x; i < blocks; i += 256) s += sums[i];
  s = block_sum_256(s, tmp);
  if (threadIdx.x != 0) return;
  const double norm = fabs(inv_scale) * sqrt(s);
  *norm_out = (float)norm;
  if (!info) return;
  const double f =
      norm > max_norm && (float)norm < INFINITY ? inv_scale * (max_norm / norm) : inv_scale;
  const bool small = fabs(f) < 0x1p-126;
  info->a = (float)(small ? f * 0x1p126 : f);
  info->b = small ? 0x1p-126f : 1.f;
}

__global__ __launch_bounds__(256) void k_scale(const TensorList L, const NormInfo *info) {
  const int t = tensor_of(L, blockIdx.x);
  const int64_t a = (int64_t)(blockIdx.x - L.first[t]) * kChunk;
  const int64_t b = a + kChunk < L.length[t] ? a + kChunk : L.length[t];
  const float fa = info->a, fb = info->b;
  by_dtype(L.dtype[t], [&](auto *p) {
    using T = std::remove_pointer_t<decltype(p)>;
    const T *x = static_cast<const T *>(L.from[t]);
    T *y = static_cast<T *>(L.to[t]);
    if (fa == 1.f && x == y) return;
    for (int64_t i = a + (int)threadIdx.x; i < b; i += 256) y[i] = (T)((float)x[i] * fa * fb);
  });
}

int blocks_of(int32_t count, const int64_t *lengths, int64_t *blocks) {
  if (count < 0 || (count > 0 && !lengths))
    return set_error(BSSCL_EINVAL, "gradient norm: null or negative list");
  int64_t n = 0;
  for (int32_t t = 0; t < count; ++t) {
    if (lengths[t] < 0) return set_error(BSSCL_EINVAL, "gradient norm: negative length");
    n += lengths[t] / kChunk + (lengths[t] % kChunk != 0);
    if (n >= kMaxBlocks) return set_error(BSSCL_EINVAL, "gradient norm: too many values");
  }
  *blocks = n;
  return BSSCL_OK;
}

constexpr int64_t kSumsAt = 256;  // behind NormInfo

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

// f(list, blocks, blocks before) for each launch's part of the tensors.
template <typename F>
int for_launches(int32_t count, const void *const *tensors, void *const *out,
                 const int64_t *lengths, const int32_t *dtypes, F &&f) {
  TensorList L;
  int64_t done = 0;
  for (int32_t t = 0; t < count;) {
    L.count = 0;
    uint32_t blocks = 0;
    for (; t < count && L.count < kPerLaunch; ++t) {
      if (lengths[t] == 0) continue;
      const int k = L.count++;
      L.from[k] = tensors[t];
      L.to[k] = out ? out[t] : nullptr;
      L.length[k] = lengths[t];
      L.dtype[k] = (uint8_t)dtypes[t];
      L.first[k] = blocks;
      blocks += (uint32_t)((lengths[t] + kChunk - 1) / kChunk);
    }
    if (L.count == 0) break;
    f(L, blocks, done);
    done += blocks;
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
  int64_t blocks = 0;
  int rc = blocks_of(count, lengths, &blocks);
  if (rc == BSSCL_OK) rc = check_list(count, tensors, out, lengths, dtypes);
  if (rc != BSSCL_OK) return rc;
  if (!std::isfinite(inv_scale))
    return set_error(BSSCL_EINVAL, "gradient norm: inv_scale must be finite");
  if (!norm || !workspace || ((uintptr_t)workspace & 255) ||
      workspace_bytes < kSumsAt + blocks * (int64_t)sizeof(double))
    return set_error(BSSCL_EINVAL,
                     "gradient norm: null norm, or a null, short or unaligned workspace");
  DeviceScope scope;
  rc = scope.enter(device);
  if (rc != BSSCL_OK) return rc;
  hipStream_t st = static_cast<hipStream_t>(stream);
  auto *info = static_cast<NormInfo *>(workspace);
  auto *sums = reinterpret_cast<double *>(static_cast<char *>(workspace) + kSumsAt);
  rc = for_launches(count, tensors, out, lengths, dtypes,
                    [&](const TensorList &L, uint32_t n, int64_t before) {
                      k_squares<<<n, 256, 0, st>>>(L, sums + before);
                    });
  if (rc != BSSCL_OK) return rc;
  k_norm<<<1, 256, 0, st>>>(sums, blocks, inv_scale, max_norm, norm, out ? info : nullptr);
  return for_launches(out ? count : 0, tensors, out, lengths, dtypes,
                      [&](const TensorList &L, uint32_t n, int64_t) {
                        k_scale<<<n, 256, 0, st>>>(L, info);
                      });
}

}  // namespace

}  // namespace bsscl

using namespace bsscl;

extern "C" {

int bsscl_grad_norm_workspace(int32_t count, const int64_t *lengths, int64_t *bytes) {
  return no_throw([&] {
    int64_t blocks = 0;
    if (!bytes) return set_error(BSSCL_EINVAL, "gradient norm: null argument");
    const int rc = blocks_of(count, lengths, &blocks);
    if (rc == BSSCL_OK) *bytes = kSumsAt + blocks * (int64_t)sizeof(double);
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
