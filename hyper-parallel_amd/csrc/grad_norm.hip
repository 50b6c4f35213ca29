// The norm of many gradients taken together, and their clipping by it.
//
//   norm = (sum |g|^p)^(1/p) over all elements of all tensors, p = 1, 2 or infinity
//   g <- round(g * min(1, max_norm / (norm + 1e-6)))
//
// Bound by memory: one read for the norm, one read and write where there is something to clip.  The tensors' table travels as a kernel argument,
// so a call can be captured and copies nothing to the GPU.  Work is dealt out by bytes: about kWorkgroups workgroups in all, whatever the tensors'
// sizes.  Sums are fp64, in which the square of any element of the three types is exact and neither overflows nor vanishes; each workgroup
// writes its own, and one workgroup adds those up in a fixed order: the same bits every time.
#include <algorithm>
#include <exception>
#include <utility>
#include <vector>

#include "hpfp8_host.h"
#include "rows.h"

namespace hpfp8 {
namespace {

constexpr int kBatch = 160;               // tensors per launch: their table is a kernel argument, of which there are 4 KB
constexpr int kThreads = 256;
constexpr int kStep = 16384;              // bytes that a workgroup takes at a time
constexpr int64_t kWorkgroups = 2048;     // for all tensors together (and at most one more for each)

enum Power { kLargest = 0, kAbsolute = 1, kSquare = 2 };

struct GradBatch {
  void* ptr[kBatch];
  int64_t numel[kBatch];
  int wg_first[kBatch + 1];               // first workgroup of tensor e
  uint8_t type[kBatch];
  int64_t per;                            // bytes of a workgroup, a multiple of kStep
  int count;
};
static_assert(sizeof(GradBatch) <= 4096 - 64, "kernel arguments");

__device__ __forceinline__ int locate(const GradBatch& b, int wg) {
  const int lane = threadIdx.x & 63;
  int e = -1;
#pragma unroll
  for (int i = 0; i < kBatch; i += 64) e += __builtin_popcountll(__ballot(i + lane < b.count && b.wg_first[i + lane < kBatch ? i + lane : 0] <= wg));
  return __builtin_amdgcn_readfirstlane(e);
}

// f(element type, first element, elements) of this workgroup's part of its tensor
template <typename F>
__device__ __forceinline__ void own_part(const GradBatch& b, F&& f) {
  const int e = locate(b, blockIdx.x), type = b.type[e];
  const int64_t per = b.per / (type == HPFP8_OUT_F32 ? 4 : 2), first = (int64_t)((int)blockIdx.x - b.wg_first[e]) * per;
  const int64_t left = b.numel[e] - first, n = left < per ? left : per;
  if (type == HPFP8_OUT_BF16) f(Bf16(), (uint16_t*)b.ptr[e] + first, n);
  else if (type == HPFP8_TYPE_F16) f(F16(), (_Float16*)b.ptr[e] + first, n);
  else f(F32(), (float*)b.ptr[e] + first, n);
}

template <int POWER>
__device__ __forceinline__ double joined(double a, double b) {
  if (POWER != kLargest) return a + b;
  return a != a || a > b ? a : b;         // (a NaN on either side stays)
}

// the workgroup's total, in thread 0
template <int POWER, int WAVES>
__device__ __forceinline__ double workgroup_total(double v) {
  __shared__ double parts[WAVES];
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) v = joined<POWER>(v, __shfl_xor(v, d));
  if ((threadIdx.x & 63) == 0) parts[threadIdx.x >> 6] = v;
  __syncthreads();
  double total = parts[0];
#pragma unroll
  for (int k = 1; k < WAVES; ++k) total = joined<POWER>(total, parts[k]);
  return total;
}

template <int POWER>
__global__ __launch_bounds__(kThreads) void grad_norm_kernel(const GradBatch b, double* __restrict__ partial) {
  double total = 0.0;
  own_part(b, [&](auto type, auto* g, int64_t n) {
    using E = decltype(type);
    constexpr int U = kStep / (kThreads * 8 * (int)sizeof(typename E::raw));
    for (int64_t at = (int64_t)threadIdx.x * 8; at < n; at += kThreads * 8 * U) {
      Pack8<E> p[U];
#pragma unroll
      for (int u = 0; u < U; ++u) p[u] = load_pack8<E, false>(g + at + u * (kThreads * 8), (int)(n - at - u * (kThreads * 8) < 8 ? n - at - u * (kThreads * 8) : 8));
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float v[8];
        unpack8<E>(p[u], v);
        if (POWER == kLargest) {
          total = joined<POWER>(total, (double)magnitude8(v));
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const double d = (double)v[i];
            total = POWER == kSquare ? __builtin_fma(d, d, total) : total + __builtin_fabs(d);
          }
        }
      }
    }
  });
  total = workgroup_total<POWER, kThreads / 64>(total);
  if (threadIdx.x == 0) partial[blockIdx.x] = total;
}

template <int POWER>
__global__ __launch_bounds__(1024) void grad_norm_finish_kernel(const double* __restrict__ partial, int64_t count, float* __restrict__ norm) {
  double total = 0.0;
  for (int64_t i = threadIdx.x; i < count; i += 1024) total = joined<POWER>(total, partial[i]);
  total = workgroup_total<POWER, 16>(total);
  if (threadIdx.x == 0) *norm = (float)(POWER == kSquare ? sqrt(total) : total);
}

__global__ __launch_bounds__(kThreads) void grad_clip_kernel(const GradBatch b, const float* __restrict__ norm, float max_norm) {
  const float factor = max_norm / (*norm + 1e-6f);
  if (factor >= 1.f) return;                // (a factor that is no number goes on)
  own_part(b, [&](auto type, auto* g, int64_t n) {
    using E = decltype(type);
    constexpr int U = kStep / (kThreads * 8 * (int)sizeof(typename E::raw));
    for (int64_t at = (int64_t)threadIdx.x * 8; at < n; at += kThreads * 8 * U) {
      Pack8<E> p[U];
      auto left = [&](int u) { return (int)(n - at - u * (kThreads * 8) < 8 ? n - at - u * (kThreads * 8) : 8); };
#pragma unroll
      for (int u = 0; u < U; ++u) p[u] = load_pack8<E>(g + at + u * (kThreads * 8), left(u));
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float v[8];
        unpack8<E>(p[u], v);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] *= factor;
        store8<E>(g + at + u * (kThreads * 8), left(u), v);
      }
    }
  });
}

int element_bytes(int type) { return type == HPFP8_OUT_F32 ? 4 : 2; }

// bytes of a workgroup
int64_t share(const int64_t* numels, const int* types, int64_t count) {
  int64_t bytes = 0;
  for (int64_t e = 0; e < count; ++e) bytes += numels[e] * element_bytes(types[e]);
  return std::max<int64_t>(1, (bytes + kWorkgroups * kStep - 1) / (kWorkgroups * kStep)) * kStep;
}
int64_t workgroups(int64_t numel, int type, int64_t per) { return (numel * element_bytes(type) + per - 1) / per; }

int check(const char* what, const void* const* ptrs, const int64_t* numels, const int* types, int64_t count) {
  HPFP8_REQUIRE(count >= 0, HPFP8_ERR_SHAPE, "%s: negative count", what);
  HPFP8_REQUIRE(count == 0 || (ptrs && numels && types), HPFP8_ERR_ARG, "%s: null table", what);
  int64_t bytes = 0;
  for (int64_t e = 0; e < count; ++e) {
    HPFP8_REQUIRE(types[e] >= 0 && types[e] <= 2, HPFP8_ERR_ARG, "%s: unknown element type %d of tensor %lld", what, types[e], (long long)e);
    HPFP8_REQUIRE(numels[e] >= 0 && numels[e] < ((int64_t)1 << 44) && bytes < ((int64_t)1 << 46), HPFP8_ERR_SHAPE, "%s: tensor %lld has %lld elements",
                  what, (long long)e, (long long)numels[e]);
    HPFP8_REQUIRE(numels[e] == 0 || ptrs[e], HPFP8_ERR_ARG, "%s: tensor %lld is null", what, (long long)e);
    HPFP8_REQUIRE(((uintptr_t)ptrs[e] & (element_bytes(types[e]) - 1)) == 0, HPFP8_ERR_ALIGN, "%s: tensor %lld is not aligned to its elements", what,
                  (long long)e);
    bytes += numels[e] * element_bytes(types[e]);
  }
  return HPFP8_OK;
}

// launch(batch, workgroups, workgroups before it) for runs of tensors
template <class F>
int for_each_batch(void* const* ptrs, const int64_t* numels, const int* types, int64_t count, F launch) {
  const int64_t per = share(numels, types, count);
  int64_t before = 0;
  for (int64_t e = 0; e < count;) {
    GradBatch b;
    b.per = per;
    b.count = 0;
    int64_t wgs = 0;
    for (; e < count && b.count < kBatch; ++e) {
      if (numels[e] == 0) continue;
      b.ptr[b.count] = ptrs[e];
      b.numel[b.count] = numels[e];
      b.type[b.count] = (uint8_t)types[e];
      b.wg_first[b.count++] = (int)wgs;
      wgs += workgroups(numels[e], types[e], per);
    }
    b.wg_first[b.count] = (int)wgs;
    if (b.count == 0) break;
    const int rc = launch(b, (unsigned)wgs, before);
    if (rc != HPFP8_OK) return rc;
    before += wgs;
  }
  return HPFP8_OK;
}

template <int POWER>
int grad_norm(const void* const* ptrs, const int64_t* numels, const int* types, int64_t count, double* partial, float* norm, hipStream_t stream) {
  const int rc = for_each_batch(const_cast<void* const*>(ptrs), numels, types, count, [&](const GradBatch& b, unsigned wgs, int64_t before) {
    grad_norm_kernel<POWER><<<wgs, kThreads, 0, stream>>>(b, partial + before);
    return check_launch("grad_norm");
  });
  if (rc != HPFP8_OK) return rc;
  grad_norm_finish_kernel<POWER><<<1, 1024, 0, stream>>>(partial, hpfp8_grad_norm_partials(numels, types, count), norm);
  return check_launch("grad_norm (finish)");
}

}  // namespace
}  // namespace hpfp8

using namespace hpfp8;

extern "C" {

int64_t hpfp8_grad_norm_partials(const int64_t* numels, const int* types, int64_t count) {
  if (count <= 0 || !numels || !types) return 0;
  const int64_t per = share(numels, types, count);
  int64_t wgs = 0;
  for (int64_t e = 0; e < count; ++e) wgs += workgroups(numels[e], types[e], per);
  return wgs;
}

int hpfp8_grad_norm(const void* const* ptrs, const int64_t* numels, const int* types, int64_t count, int power, double* partial, float* norm,
                    hpfp8_stream_t stream) {
  const int rc = check("grad_norm", ptrs, numels, types, count);
  if (rc != HPFP8_OK) return rc;
  HPFP8_REQUIRE(power >= kLargest && power <= kSquare, HPFP8_ERR_ARG, "grad_norm: the power must be 1, 2 or 0 for infinity, got %d", power);
  HPFP8_REQUIRE(norm && (partial || hpfp8_grad_norm_partials(numels, types, count) == 0), HPFP8_ERR_ARG, "grad_norm: null buffer");
  if (power == kLargest) return grad_norm<kLargest>(ptrs, numels, types, count, partial, norm, (hipStream_t)stream);
  if (power == kAbsolute) return grad_norm<kAbsolute>(ptrs, numels, types, count, partial, norm, (hipStream_t)stream);
  return grad_norm<kSquare>(ptrs, numels, types, count, partial, norm, (hipStream_t)stream);
}

int hpfp8_grad_clip(void* const* ptrs, const int64_t* numels, const int* types, int64_t count, const float* norm, float max_norm,
                    hpfp8_stream_t stream) {
  int rc = check("grad_clip", ptrs, numels, types, count);
  if (rc != HPFP8_OK) return rc;
  HPFP8_REQUIRE(norm || count == 0, HPFP8_ERR_ARG, "grad_clip: null norm");
  // memory that two tensors share would be read and written twice at once
  try {
    std::vector<std::pair<uintptr_t, uintptr_t>> spans;
    spans.reserve(count);
    for (int64_t e = 0; e < count; ++e)
      if (numels[e] > 0) spans.emplace_back((uintptr_t)ptrs[e], (uintptr_t)ptrs[e] + numels[e] * element_bytes(types[e]));
    std::sort(spans.begin(), spans.end());
    for (size_t i = 1; i < spans.size(); ++i)
      HPFP8_REQUIRE(spans[i].first >= spans[i - 1].second, HPFP8_ERR_ARG, "grad_clip: two tensors share memory");
  } catch (const std::exception&) {
    return fail(HPFP8_ERR_ARG, "grad_clip: no memory for a table of %lld tensors", (long long)count);
  }
  return for_each_batch(ptrs, numels, types, count, [&](const GradBatch& b, unsigned wgs, int64_t) {
    grad_clip_kernel<<<wgs, kThreads, 0, (hipStream_t)stream>>>(b, norm, max_norm);
    return check_launch("grad_clip");
  });
}

}  // extern "C"
