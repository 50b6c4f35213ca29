// The norm of many gradients taken together, and their clipping by it.
//
//   norm = (sum |g|^p)^(1/p) over all elements of all tensors, p = 1, 2 or infinity
//   g <- round(g * min(1, max_norm / (norm + 1e-6)))
//
// Bound by memory: one read for the norm, one read and write where there is something to clip.  The tensors' table travels as a kernel argument,
// so a call can be captured and copies nothing to the GPU.  Work is dealt out by bytes, whatever the tensors' sizes: the norm in about
// kNormParts parts, the clipping in parts of 16 KB.  Sums are fp64, in which the square of any element of the three types is exact and neither
// overflows nor vanishes; each workgroup writes its own, and they are added up in a fixed order: the same bits every time.
// Tensors of more than the Infinity Cache together (256 MiB) are streamed past the caches, and one workgroup clips one part: 2 GiB of fp32 read at
// 6.9 TB/s, where ordinary loads reach 6.1, and read and written at 6.0, where 2048 workgroups that go through them reach 5.2.  (Parts of 4 KB
// reach 6.6, but where the bound holds 524288 workgroups take 114 us to find that there is nothing to do, 131072 take 31.)  Of smaller ones the
// second pass finds in the caches what the first has read (140 MiB read and written at 7.7 TB/s, streamed 6.1), and where the bound holds its 256
// workgroups of 1024 threads end in 4 to 5 us, the sums' addition among them.
#include <algorithm>
#include <exception>
#include <type_traits>
#include <utility>
#include <vector>

#include "hpfp8_host.h"
#include "rows.h"

namespace hpfp8 {
namespace {

constexpr int kBatch = 250;               // tensors per launch: their table is a kernel argument, of which there are 4 KB
constexpr int kThreads = 256;
constexpr int kStep = 16384;              // bytes that a workgroup takes at a time
constexpr int64_t kNormParts = 8192;      // for all tensors together (and at most one more for each)
constexpr int64_t kCached = (int64_t)256 << 20;
constexpr unsigned kClipWorkgroups = 1024;

enum Power { kLargest = 0, kAbsolute = 1, kSquare = 2 };

// A tensor is two words: its address with its element type above, and its first part (kPartBits) with its elements above.
constexpr int kTypeShift = 56, kPartBits = 27;
constexpr int64_t kMostElements = (int64_t)1 << (64 - kPartBits), kMostBytes = (int64_t)1 << 40;      // (so that all parts of 16 KB are counted in kPartBits)
struct GradBatch {
  uint64_t where[kBatch], what[kBatch];
  int64_t per;                            // bytes of a part, a multiple of kStep
  int count, parts;
};
static_assert(sizeof(GradBatch) <= 4096 - 64, "kernel arguments");
static_assert((kMostBytes / kStep + (1 << 20)) >> kPartBits == 0, "first parts");

__device__ __forceinline__ int locate(const GradBatch& b, int part) {
  const int lane = threadIdx.x & 63;
  int e = -1;
#pragma unroll
  for (int i = 0; i < kBatch; i += 64)
    e += __builtin_popcountll(__ballot(i + lane < b.count && (int)(b.what[i + lane < kBatch ? i + lane : 0] & ((1 << kPartBits) - 1)) <= part));
  return __builtin_amdgcn_readfirstlane(e);
}

// A part of the tensors as memory: units of 16 bits, of which an fp32 has two.
struct Part {
  uint16_t* at;
  int64_t units;
  int type;
};
__device__ __forceinline__ Part part_of(const GradBatch& b, int part) {
  const int e = locate(b, part);
  const uint64_t where = b.where[e], what = b.what[e];
  const int type = (int)(where >> kTypeShift);
  const int64_t first = (int64_t)(part - (int)(what & ((1 << kPartBits) - 1))) * (b.per / 2);
  const int64_t left = (int64_t)(what >> kPartBits) * (type == HPFP8_OUT_F32 ? 2 : 1) - first;
  return {(uint16_t*)(where & (((uint64_t)1 << kTypeShift) - 1)) + first, left < b.per / 2 ? left : b.per / 2, type};
}

template <int POWER>
__device__ __forceinline__ double joined(double a, double b) {
  if (POWER != kLargest) return a + b;
  return a != a || a > b ? a : b;         // (a NaN on either side stays)
}

template <int POWER>
__device__ __forceinline__ double wave_joined(double v) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) v = joined<POWER>(v, __shfl_xor(v, d));
  return v;
}

// Sixteen neighbouring bytes from any element on, n units of them there (8 or more: all; 0 or less: none), the others zeros.  WHOLE: all are there.
template <bool STREAM, bool WHOLE>
__device__ __forceinline__ u32x4 load16(const uint16_t* p, int64_t n) {
  if (WHOLE || n >= 8) {
    const u32x4_at2* q = reinterpret_cast<const u32x4_at2*>(p);
    return STREAM ? __builtin_nontemporal_load(q) : *q;
  }
  u32x4 w = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < n) w[i / 2] |= (uint32_t)p[i] << (16 * (i % 2));
  return w;
}
template <bool STREAM, bool WHOLE>
__device__ __forceinline__ void store16(uint16_t* p, int64_t n, const u32x4& w) {
  if (WHOLE || n >= 8) {
    u32x4_at2* q = reinterpret_cast<u32x4_at2*>(p);
    if (STREAM) __builtin_nontemporal_store((u32x4_at2)w, q);
    else *q = w;
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < n) p[i] = (uint16_t)(w[i / 2] >> (16 * (i % 2)));
}
template <typename E>
constexpr int kPer = 16 / (int)sizeof(typename E::raw);       // elements of 16 bytes
template <typename E>
__device__ __forceinline__ void values16(const u32x4& w, float v[8]) {
  if constexpr (kPer<E> == 8) {
    Pack8<E> p;
    p.w[0] = w;
    unpack8<E>(p, v);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(w[i]);
  }
}
template <typename F>
__device__ __forceinline__ void by_type(int type, F&& f) {
  if (type == HPFP8_OUT_BF16) f(Bf16());
  else if (type == HPFP8_TYPE_F16) f(F16());
  else f(F32());
}
constexpr int U = kStep / (kThreads * 16);                     // vectors of a thread and step
template <bool STREAM, bool WHOLE>
__device__ __forceinline__ void load_step(const Part& p, int64_t at, u32x4 w[U]) {
#pragma unroll
  for (int u = 0; u < U; ++u) w[u] = load16<STREAM, WHOLE>(p.at + at + u * (kThreads * 8), p.units - at - u * (kThreads * 8));
}

template <int POWER, bool STREAM>
__global__ __launch_bounds__(kThreads) void grad_norm_kernel(const GradBatch b, double* __restrict__ partial) {
  double total = 0.0;
  const Part p = part_of(b, blockIdx.x);
  by_type(p.type, [&](auto type) {
    using E = decltype(type);
    auto step = [&](int64_t at, auto whole) {
      u32x4 w[U];
      load_step<STREAM, whole>(p, at, w);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float v[8];
        values16<E>(w[u], v);
#pragma unroll
        for (int i = 0; i < kPer<E>; ++i) {
          if (POWER == kLargest) {
            total = joined<POWER>(total, (double)__builtin_fabsf(v[i]));
          } else {
            const double d = (double)v[i];
            total = POWER == kSquare ? __builtin_fma(d, d, total) : total + __builtin_fabs(d);
          }
        }
      }
    };
    constexpr int kUnits = kStep / 2;
    const int64_t whole = p.units / kUnits * kUnits, mine = threadIdx.x * 8;
    for (int64_t at = 0; at < whole; at += kUnits) step(at + mine, std::true_type());
    if (whole < p.units) step(whole + mine, std::false_type());
  });
  __shared__ double parts[kThreads / 64];
  total = wave_joined<POWER>(total);
  if ((threadIdx.x & 63) == 0) parts[threadIdx.x >> 6] = total;
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int k = 1; k < kThreads / 64; ++k) total = joined<POWER>(total, parts[k]);
    partial[blockIdx.x] = total;
  }
}

// the norm, from the workgroups' sums, by one workgroup of 1024 threads
template <int POWER>
__device__ __forceinline__ float finished(const double* __restrict__ partial, int64_t count) {
  __shared__ double parts[16];
  double total = 0.0;
  for (int64_t i = threadIdx.x; i < count; i += 1024) total = joined<POWER>(total, partial[i]);
  total = wave_joined<POWER>(total);
  if ((threadIdx.x & 63) == 0) parts[threadIdx.x >> 6] = total;
  __syncthreads();
  total = parts[0];
#pragma unroll
  for (int k = 1; k < 16; ++k) total = joined<POWER>(total, parts[k]);
  return (float)(POWER == kSquare ? sqrt(total) : total);
}

template <int POWER>
__global__ __launch_bounds__(1024) void grad_norm_finish_kernel(const double* __restrict__ partial, int64_t count, float* __restrict__ norm) {
  const float total = finished<POWER>(partial, count);
  if (threadIdx.x == 0) *norm = total;
}

// A part to clip is one step.
template <bool STREAM>
__device__ __forceinline__ void load_part(const Part& p, u32x4 w[U]) {
  const int64_t at = threadIdx.x % kThreads * 8;
  if (p.units == kStep / 2) load_step<STREAM, true>(p, at, w);
  else load_step<STREAM, false>(p, at, w);
}
template <bool STREAM>
__device__ __forceinline__ void clip_part(const Part& p, u32x4 w[U], float factor) {
  const int64_t at = threadIdx.x % kThreads * 8;
  by_type(p.type, [&](auto type) {
    using E = decltype(type);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float v[8];
      values16<E>(w[u], v);
#pragma unroll
      for (int i = 0; i < kPer<E>; ++i) v[i] *= factor;
      if constexpr (kPer<E> == 8) {
        w[u] = pack8<E>(v).w[0];
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) w[u][i] = __float_as_uint(v[i]);
      }
    }
  });
  if (p.units == kStep / 2) {
#pragma unroll
    for (int u = 0; u < U; ++u) store16<STREAM, true>(p.at + at + u * (kThreads * 8), 8, w[u]);
  } else {
#pragma unroll
    for (int u = 0; u < U; ++u) store16<STREAM, false>(p.at + at + u * (kThreads * 8), p.units - at - u * (kThreads * 8), w[u]);
  }
}

__device__ __forceinline__ float clip_factor(float norm, float max_norm) { return max_norm / (norm + 1e-6f); }

// One part per workgroup, or the parts one after the other (a factor that is no number goes on).
template <bool STREAM>
__global__ __launch_bounds__(kThreads) void grad_clip_kernel(const GradBatch b, const float* __restrict__ norm, float max_norm) {
  const float factor = clip_factor(*norm, max_norm);
  if (factor >= 1.f) return;
  for (int part = blockIdx.x; part < b.parts; part += gridDim.x) {
    const Part p = part_of(b, part);
    u32x4 w[U];
    load_part<STREAM>(p, w);
    clip_part<STREAM>(p, w, factor);
  }
}

// Behind the norm's kernel: every workgroup adds its sums up, in the same order, which is shorter than a launch for that; where
// there is one part for each of its quarters, that is under way meanwhile.  (With 256 threads the sums of 8192 parts took 10 us, so 4.)
template <int POWER>
__global__ __launch_bounds__(1024) void grad_finish_and_clip_kernel(const GradBatch b, const double* __restrict__ partial, int64_t count,
                                                                    float* __restrict__ norm, float max_norm) {
  constexpr int kQuarters = 1024 / kThreads;
  int part = blockIdx.x * kQuarters + __builtin_amdgcn_readfirstlane(threadIdx.x / kThreads);
  const int parts = b.parts;
  Part p = {nullptr, 0, 0};
  u32x4 w[U];
  const bool once = parts <= (int)gridDim.x * kQuarters;       // (of more, the first parts would be a fifth of all, read for nothing where the bound holds)
  if (once && part < parts) p = part_of(b, part);
  load_part<false>(p, w);
  const float total = finished<POWER>(partial, count);
  if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = total;
  const float factor = clip_factor(total, max_norm);
  if (factor >= 1.f) return;
  for (; part < parts; part += gridDim.x * kQuarters) {
    if (!once) {
      p = part_of(b, part);
      load_part<false>(p, w);
    }
    clip_part<false>(p, w, factor);
  }
}

int element_bytes(int type) { return type == HPFP8_OUT_F32 ? 4 : 2; }

int64_t all_bytes(const int64_t* numels, const int* types, int64_t count) {
  int64_t bytes = 0;
  for (int64_t e = 0; e < count; ++e) bytes += numels[e] * element_bytes(types[e]);
  return bytes;
}
// bytes of a workgroup of the norm
int64_t norm_part(int64_t bytes) { return std::max<int64_t>(1, (bytes + kNormParts * kStep - 1) / (kNormParts * kStep)) * kStep; }
int64_t parts_of(int64_t numel, int type, int64_t per) { return (numel * element_bytes(type) + per - 1) / per; }

int check(const char* what, const void* const* ptrs, const int64_t* numels, const int* types, int64_t count) {
  HPFP8_REQUIRE(count >= 0, HPFP8_ERR_SHAPE, "%s: negative count", what);
  HPFP8_REQUIRE(count == 0 || (ptrs && numels && types), HPFP8_ERR_ARG, "%s: null table", what);
  int64_t bytes = 0;
  for (int64_t e = 0; e < count; ++e) {
    HPFP8_REQUIRE(types[e] >= 0 && types[e] <= 2, HPFP8_ERR_ARG, "%s: unknown element type %d of tensor %lld", what, types[e], (long long)e);
    HPFP8_REQUIRE(numels[e] >= 0 && numels[e] < kMostElements && bytes < kMostBytes, HPFP8_ERR_SHAPE, "%s: tensor %lld has %lld elements",
                  what, (long long)e, (long long)numels[e]);
    HPFP8_REQUIRE(numels[e] == 0 || ptrs[e], HPFP8_ERR_ARG, "%s: tensor %lld is null", what, (long long)e);
    HPFP8_REQUIRE((uint64_t)(uintptr_t)ptrs[e] >> kTypeShift == 0, HPFP8_ERR_ARG, "%s: tensor %lld has no address of this machine", what, (long long)e);
    HPFP8_REQUIRE(((uintptr_t)ptrs[e] & (element_bytes(types[e]) - 1)) == 0, HPFP8_ERR_ALIGN, "%s: tensor %lld is not aligned to its elements", what,
                  (long long)e);
    bytes += numels[e] * element_bytes(types[e]);
  }
  HPFP8_REQUIRE(bytes < kMostBytes, HPFP8_ERR_SHAPE, "%s: %lld bytes", what, (long long)bytes);
  return HPFP8_OK;
}

// launch(batch, parts, parts before it) for runs of tensors; per: bytes of a part
template <class F>
int for_each_batch(const void* const* ptrs, const int64_t* numels, const int* types, int64_t count, int64_t per, F launch) {
  int64_t before = 0;
  for (int64_t e = 0; e < count;) {
    GradBatch b;
    b.per = per;
    b.count = 0;
    int64_t parts = 0;
    for (; e < count && b.count < kBatch; ++e) {
      if (numels[e] == 0) continue;
      b.where[b.count] = (uint64_t)(uintptr_t)ptrs[e] | (uint64_t)types[e] << kTypeShift;
      b.what[b.count++] = (uint64_t)parts | (uint64_t)numels[e] << kPartBits;
      parts += parts_of(numels[e], types[e], per);
    }
    b.parts = (int)parts;
    if (b.count == 0) break;
    const int rc = launch(b, (unsigned)parts, before);
    if (rc != HPFP8_OK) return rc;
    before += parts;
  }
  return HPFP8_OK;
}

int clip(void* const* ptrs, const int64_t* numels, const int* types, int64_t count, const float* norm, float max_norm, hipStream_t stream) {
  const bool streamed = all_bytes(numels, types, count) > kCached;
  return for_each_batch(ptrs, numels, types, count, kStep, [&](const GradBatch& b, unsigned parts, int64_t) {
    if (streamed) grad_clip_kernel<true><<<std::min(parts, 1u << 22), kThreads, 0, stream>>>(b, norm, max_norm);
    else grad_clip_kernel<false><<<std::min(parts, kClipWorkgroups), kThreads, 0, stream>>>(b, norm, max_norm);
    return check_launch("grad_clip");
  });
}

// max_norm: negative for the norm alone
template <int POWER>
int grad_norm(void* const* ptrs, const int64_t* numels, const int* types, int64_t count, double* partial, float* norm, float max_norm,
              hipStream_t stream) {
  const int64_t bytes = all_bytes(numels, types, count), sums = hpfp8_grad_norm_partials(numels, types, count);
  int rc = for_each_batch(ptrs, numels, types, count, norm_part(bytes), [&](const GradBatch& b, unsigned parts, int64_t before) {
    if (bytes > kCached) grad_norm_kernel<POWER, true><<<parts, kThreads, 0, stream>>>(b, partial + before);
    else grad_norm_kernel<POWER, false><<<parts, kThreads, 0, stream>>>(b, partial + before);
    return check_launch("grad_norm");
  });
  if (rc != HPFP8_OK) return rc;
  if (max_norm >= 0.f && bytes > 0 && bytes <= kCached)
    return for_each_batch(ptrs, numels, types, count, kStep, [&](const GradBatch& b, unsigned parts, int64_t before) {
      grad_finish_and_clip_kernel<POWER><<<std::min((parts + 3) / 4, kClipWorkgroups / 4), 1024, 0, stream>>>(b, partial, sums, before ? nullptr : norm, max_norm);
      return check_launch("grad_norm_and_clip");
    });
  grad_norm_finish_kernel<POWER><<<1, 1024, 0, stream>>>(partial, sums, norm);
  rc = check_launch("grad_norm (finish)");
  return rc != HPFP8_OK || max_norm < 0.f ? rc : clip(ptrs, numels, types, count, norm, max_norm, stream);
}

int by_power(const char* what, void* const* ptrs, const int64_t* numels, const int* types, int64_t count, int power, double* partial, float* norm,
             float max_norm, hipStream_t stream) {
  HPFP8_REQUIRE(power >= kLargest && power <= kSquare, HPFP8_ERR_ARG, "%s: the power must be 1, 2 or 0 for infinity, got %d", what, power);
  HPFP8_REQUIRE(norm && (partial || hpfp8_grad_norm_partials(numels, types, count) == 0), HPFP8_ERR_ARG, "%s: null buffer", what);
  if (power == kLargest) return grad_norm<kLargest>(ptrs, numels, types, count, partial, norm, max_norm, stream);
  if (power == kAbsolute) return grad_norm<kAbsolute>(ptrs, numels, types, count, partial, norm, max_norm, stream);
  return grad_norm<kSquare>(ptrs, numels, types, count, partial, norm, max_norm, stream);
}

// memory that two tensors share would be read and written twice at once
int check_apart(const char* what, const void* const* ptrs, const int64_t* numels, const int* types, int64_t count) {
  try {
    std::vector<std::pair<uintptr_t, uintptr_t>> spans;
    spans.reserve(count);
    for (int64_t e = 0; e < count; ++e)
      if (numels[e] > 0) spans.emplace_back((uintptr_t)ptrs[e], (uintptr_t)ptrs[e] + numels[e] * element_bytes(types[e]));
    std::sort(spans.begin(), spans.end());
    for (size_t i = 1; i < spans.size(); ++i)
      HPFP8_REQUIRE(spans[i].first >= spans[i - 1].second, HPFP8_ERR_ARG, "%s: two tensors share memory", what);
  } catch (const std::exception&) {
    return fail(HPFP8_ERR_ARG, "%s: no memory for a table of %lld tensors", what, (long long)count);
  }
  return HPFP8_OK;
}

}  // namespace
}  // namespace hpfp8

using namespace hpfp8;

extern "C" {

int64_t hpfp8_grad_norm_partials(const int64_t* numels, const int* types, int64_t count) {
  if (count <= 0 || !numels || !types) return 0;
  const int64_t per = norm_part(all_bytes(numels, types, count));
  int64_t parts = 0;
  for (int64_t e = 0; e < count; ++e) parts += parts_of(numels[e], types[e], per);
  return parts;
}

int hpfp8_grad_norm(const void* const* ptrs, const int64_t* numels, const int* types, int64_t count, int power, double* partial, float* norm,
                    hpfp8_stream_t stream) {
  const int rc = check("grad_norm", ptrs, numels, types, count);
  return rc != HPFP8_OK ? rc : by_power("grad_norm", const_cast<void* const*>(ptrs), numels, types, count, power, partial, norm, -1.f, (hipStream_t)stream);
}

int hpfp8_grad_norm_and_clip(void* const* ptrs, const int64_t* numels, const int* types, int64_t count, int power, float max_norm, double* partial,
                             float* norm, hpfp8_stream_t stream) {
  const char* what = "grad_norm_and_clip";
  int rc = check(what, ptrs, numels, types, count);
  if (rc != HPFP8_OK) return rc;
  HPFP8_REQUIRE(max_norm >= 0.f, HPFP8_ERR_ARG, "%s: a negative bound", what);
  rc = check_apart(what, ptrs, numels, types, count);
  return rc != HPFP8_OK ? rc : by_power(what, ptrs, numels, types, count, power, partial, norm, max_norm, (hipStream_t)stream);
}

int hpfp8_grad_clip(void* const* ptrs, const int64_t* numels, const int* types, int64_t count, const float* norm, float max_norm,
                    hpfp8_stream_t stream) {
  int rc = check("grad_clip", ptrs, numels, types, count);
  if (rc != HPFP8_OK) return rc;
  HPFP8_REQUIRE(norm || count == 0, HPFP8_ERR_ARG, "grad_clip: null norm");
  rc = check_apart("grad_clip", ptrs, numels, types, count);
  if (rc != HPFP8_OK) return rc;
  return clip(ptrs, numels, types, count, norm, max_norm, (hipStream_t)stream);
}

}  // extern "C"
