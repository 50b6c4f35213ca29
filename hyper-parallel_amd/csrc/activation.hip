// Activations kept in 8 bits: a tensor's E4M3 codes with one fp32 scale for each 128 values of a row (the last group of a row is what
// is left of it), made and read back by themselves, and inside the forward and the backward of silu, gelu and SwiGLU.
//
// All four kernels are one pass over memory and bound by it: bytes per value, bf16, quantize 2 + 1.03, read back 1.03 + 2, forward of an
// ungated activation 2 + 2 + 1.03, its backward 2 + 1.03 + 2 (SwiGLU, per value of the gate/up pair: 2 + 1 + 1.03 and 1 + 1.03 + 2).
// Sixteen lanes own one scaling group, eight values each, so a group's maximum is four steps across lanes and its codes leave as 128
// bytes.  A workgroup is 16 such groups, next to each other along a row as far as the row goes and then down the rows, and takes
// kUnroll row steps with all their loads in flight.
//
// bf16, 16384 x 7168: quantize 58 us, 6.1 TB/s, read back 60 us, 5.9 TB/s (with the codes for infinities and NaN 60 and 60); SwiGLU, 4096 x 36864: forward 102 us, backward 100 us, 6.0 TB/s.
#include <type_traits>

#include "hpfp8_host.h"
#include "rows.h"

namespace hpfp8 {
namespace {

constexpr int kUnroll = 4;
enum Kind { kSilu = 0, kGelu = 1, kGeluTanh = 2, kSwiglu = 3 };

// ---- the functions and their derivatives, in fp32
// 1 / (1 + exp(-x)): the hardware's base-2 exponential and reciprocal, each within one unit in the last place; 0 below 2^-126 (x < -87).
__device__ __forceinline__ float sigmoid(float x) { return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x * -1.44269504f)); }

// The normal distribution's Phi(-a) for 0 <= a <= kFar is erfcx(a / sqrt 2) exp(-a^2 / 2) / 2, where the scaled complementary error function
// erfcx(z) is t P(t), t = 1 / (1 + 0.4 z), with a polynomial of degree 8 fitted to it on t in [0, 1] (least squares, reweighted to equal
// ripple: 1.3e-7 relative, 4.5e-7 in fp32; the factor 1 / 2 is in its coefficients).  The tail keeps its relative precision, which
// 1 + erf would lose, and the exponential is the density's too.
constexpr float kFar = 30.0f;             // (exp(-a^2 / 2) has been 0 for long)
__device__ __forceinline__ float normal_tail(float a, float& e) {
  e = __builtin_amdgcn_exp2f(a * a * -0.72134752f);             // exp(-a^2 / 2)
  const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(a, 0.28284271f, 1.0f));
  float r = 0.025132825598120689f;
  r = __builtin_fmaf(r, t, -0.091457799077034f);
  r = __builtin_fmaf(r, t, 0.0845542922616005f);
  r = __builtin_fmaf(r, t, -0.00281374366022646425f);
  r = __builtin_fmaf(r, t, 0.07072056084871292f);
  r = __builtin_fmaf(r, t, 0.084269682317972183f);
  r = __builtin_fmaf(r, t, 0.10392154008150101f);
  r = __builtin_fmaf(r, t, 0.11283478885889053f);
  r = __builtin_fmaf(r, t, 0.11283793300390244f);
  return r * t * e;
}

// x times a factor in [0, 1] that goes to zero faster than x grows: 0 for x = -inf, where the product would be NaN
__device__ __forceinline__ float damped(float x, float factor) { return factor == 0.f ? 0.f : x * factor; }

template <int KIND>
__device__ __forceinline__ float value(float x) {
  if constexpr (KIND == kSilu) return damped(x, sigmoid(x));
  if constexpr (KIND == kGelu) {
    // x Phi(x) = max(x, 0) - |x| Phi(-|x|); a NaN comes through the maximum
    const float a = fminf(fabsf(x), kFar);
    float e;
    return __builtin_elementwise_maximum(x, 0.f) - a * normal_tail(a, e);
  }
  // 0.5 x (1 + tanh(u)) = x sigmoid(2 u), u = sqrt(2 / pi) (x + 0.044715 x^3)
  return damped(x, sigmoid(x * __builtin_fmaf(x * x, 0.07135481f, 1.59576912f)));
}
template <int KIND>
__device__ __forceinline__ float derivative(float x) {
  if constexpr (KIND == kGelu) {
    const float near = __builtin_elementwise_maximum(__builtin_elementwise_minimum(x, kFar), -kFar);
    float e;
    const float tail = normal_tail(fabsf(near), e), phi = x < 0.f ? tail : 1.0f - tail;
    return __builtin_fmaf(near * 0.39894228f, e, phi);
  }
  const float x2 = x * x;
  const float s = KIND == kSilu ? sigmoid(x) : sigmoid(x * __builtin_fmaf(x2, 0.07135481f, 1.59576912f));
  const float slope = s * (1.0f - s);
  const float inner = KIND == kSilu ? x : x * __builtin_fmaf(x2, 0.21406444f, 1.59576912f);   // x d(2 u)/dx
  return s + damped(inner, slope);
}

// ---- where a group of 16 lanes is
struct Grid {
  int64_t rows;
  int64_t cols;        // of one half, for SwiGLU
  int groups;          // of a row (of one half): cols / 128 rounded up
  int across;          // groups of a workgroup along a row: 1, 2, 4, 8 or 16
};

struct Place {
  int64_t row, step;   // first row, and rows from one of the kUnroll steps to the next
  int64_t stride;      // rows from one pass of the grid to the next
  int group;
  int64_t col;         // of this lane's eight values
  int left;            // how many there are from there on, up to eight
};

__device__ __forceinline__ Place place(const Grid& g) {
  const int l = threadIdx.x & 15, q = threadIdx.x >> 4;
  const int shift = __builtin_ctz(g.across);
  Place p;
  const int down = 16 >> shift;
  p.group = (int)blockIdx.x * g.across + (q & (g.across - 1));
  p.row = (int64_t)blockIdx.y * (down * kUnroll) + (q >> shift);
  p.step = down;
  p.stride = (int64_t)gridDim.y * (down * kUnroll);
  p.col = (int64_t)p.group * kBlock + l * 8;
  p.left = p.group < g.groups ? (int)(g.cols - p.col < 8 ? g.cols - p.col : 8) : 0;
  return p;
}

// ---- quantize and read back.  SPECIAL: infinities and NaN come back as they were and leave their group's other values alone
template <typename E, bool SPECIAL>
__global__ __launch_bounds__(256) void quantize_rows_kernel(const typename E::raw* __restrict__ x, int64_t ld, Grid g, uint8_t* __restrict__ q,
                                                            float* __restrict__ scale_inv) {
  const Place p = place(g);
  for (int64_t first = p.row; first < g.rows; first += p.stride) {
    Pack8<E> v[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int64_t r = first + u * p.step;
      v[u] = load_pack8<E>(x + (r < g.rows ? r * ld + p.col : 0), r < g.rows ? p.left : 0);
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int64_t r = first + u * p.step;
      float f[8], s;
      unpack8<E>(v[u], f);
      const uint2 c = encode_group<SPECIAL>(f, s);
      if (r < g.rows && p.left > 0) {
        store_codes8(q + r * g.cols + p.col, p.left, c);
        if ((threadIdx.x & 15) == 0) scale_inv[r * g.groups + p.group] = s;
      }
    }
  }
}

template <typename E, bool SPECIAL>
__global__ __launch_bounds__(256) void dequantize_rows_kernel(const uint8_t* __restrict__ q, const float* __restrict__ scale_inv, Grid g,
                                                              typename E::raw* __restrict__ x) {
  const Place p = place(g);
  for (int64_t first = p.row; first < g.rows; first += p.stride) {
    uint2 c[kUnroll];
    float s[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int64_t r = first + u * p.step;
      const bool in = r < g.rows && p.left > 0;
      c[u] = load_codes8(q + (in ? r * g.cols + p.col : 0), in ? p.left : 0);
      s[u] = in ? scale_inv[r * g.groups + p.group] : 0.f;
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int64_t r = first + u * p.step;
      if (r >= g.rows || p.left <= 0) break;
      float f[8];
      decode8<SPECIAL>(c[u], s[u], f);
      store8<E>(x + r * g.cols + p.col, p.left, f);
    }
  }
}

// ---- y = f(x) and x's codes (if they are kept) from one read of x; SwiGLU: x = gate | up, each half with groups of its own
template <typename E, int KIND, bool KEEP>
__global__ __launch_bounds__(256) void activation_forward_kernel(const typename E::raw* __restrict__ x, int64_t ld, Grid g,
                                                                 typename E::raw* __restrict__ y, uint8_t* __restrict__ q,
                                                                 float* __restrict__ scale_inv) {
  constexpr int kHalves = KIND == kSwiglu ? 2 : 1;
  constexpr int kSteps = KIND == kSwiglu ? kUnroll / 2 : kUnroll;
  const Place p = place(g);
  const int l = threadIdx.x & 15;
  for (int64_t first = p.row; first < g.rows; first += p.stride) {
#pragma unroll
    for (int u0 = 0; u0 < kUnroll; u0 += kSteps) {
      Pack8<E> v[kSteps][kHalves];
#pragma unroll
      for (int u = 0; u < kSteps; ++u) {
        const int64_t r = first + (u0 + u) * p.step;
#pragma unroll
        for (int h = 0; h < kHalves; ++h)
          v[u][h] = load_pack8<E>(x + (r < g.rows ? r * ld + h * g.cols + p.col : 0), r < g.rows ? p.left : 0);
      }
#pragma unroll
      for (int u = 0; u < kSteps; ++u) {
        const int64_t r = first + (u0 + u) * p.step;
        const bool in = r < g.rows && p.left > 0;
        float f[kHalves][8], out[8];
#pragma unroll
        for (int h = 0; h < kHalves; ++h) {
          unpack8<E>(v[u][h], f[h]);
          if constexpr (KEEP) {
            float s;
            const uint2 c = encode_group(f[h], s);
            if (in) {
              store_codes8(q + (r * kHalves + h) * g.cols + p.col, p.left, c);
              if (l == 0) scale_inv[(r * kHalves + h) * g.groups + p.group] = s;
            }
          }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) out[i] = KIND == kSwiglu ? value<kSilu>(f[0][i]) * f[kHalves - 1][i] : value<KIND == kSwiglu ? kSilu : KIND>(f[0][i]);
        if (in) store8<E>(y + r * g.cols + p.col, p.left, out);
      }
    }
  }
}

// ---- dx = dy f'(x), x from its codes (KEEP) or as it was
template <typename E, int KIND, bool KEEP>
__global__ __launch_bounds__(256) void activation_backward_kernel(const typename E::raw* __restrict__ dy, const typename E::raw* __restrict__ x,
                                                                  int64_t ld, const uint8_t* __restrict__ q,
                                                                  const float* __restrict__ scale_inv, Grid g,
                                                                  typename E::raw* __restrict__ dx) {
  constexpr int kHalves = KIND == kSwiglu ? 2 : 1;
  constexpr int kSteps = KIND == kSwiglu ? kUnroll / 2 : kUnroll;
  const Place p = place(g);
  for (int64_t first = p.row; first < g.rows; first += p.stride) {
#pragma unroll
    for (int u0 = 0; u0 < kUnroll; u0 += kSteps) {
      Pack8<E> d[kSteps], v[KEEP ? 1 : kSteps][kHalves];
      uint2 c[kSteps][kHalves];
      float s[kSteps][kHalves];
#pragma unroll
      for (int u = 0; u < kSteps; ++u) {
        const int64_t r = first + (u0 + u) * p.step;
        const bool in = r < g.rows && p.left > 0;
        d[u] = load_pack8<E>(dy + (in ? r * g.cols + p.col : 0), in ? p.left : 0);
#pragma unroll
        for (int h = 0; h < kHalves; ++h) {
          if constexpr (KEEP) {
            c[u][h] = load_codes8(q + (in ? (r * kHalves + h) * g.cols + p.col : 0), in ? p.left : 0);
            s[u][h] = in ? scale_inv[(r * kHalves + h) * g.groups + p.group] : 0.f;
          } else {
            v[u][h] = load_pack8<E>(x + (in ? r * ld + h * g.cols + p.col : 0), in ? p.left : 0);
          }
        }
      }
#pragma unroll
      for (int u = 0; u < kSteps; ++u) {
        const int64_t r = first + (u0 + u) * p.step;
        if (r >= g.rows || p.left <= 0) break;
        float f[kHalves][8], go[8], out[8];
        unpack8<E>(d[u], go);
#pragma unroll
        for (int h = 0; h < kHalves; ++h) {
          if constexpr (KEEP) decode8(c[u][h], s[u][h], f[h]);
          else unpack8<E>(v[u][h], f[h]);
        }
        if constexpr (KIND == kSwiglu) {
          // d gate = dy up silu'(gate), d up = dy silu(gate)
#pragma unroll
          for (int i = 0; i < 8; ++i) out[i] = go[i] * f[1][i] * derivative<kSilu>(f[0][i]);
          store8<E>(dx + r * 2 * g.cols + p.col, p.left, out);
#pragma unroll
          for (int i = 0; i < 8; ++i) out[i] = go[i] * value<kSilu>(f[0][i]);
          store8<E>(dx + (r * 2 + 1) * g.cols + p.col, p.left, out);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) out[i] = go[i] * derivative<KIND>(f[0][i]);
          store8<E>(dx + r * g.cols + p.col, p.left, out);
        }
      }
    }
  }
}

// The workgroup's shape: as many groups along a row as leave at most a quarter of them idle (rows of 8200 values with one group of each of
// 16 rows, which leaves none idle: 141 us where eight take 69).
bool shape(int64_t rows, int64_t cols, Grid& g, dim3& grid) {
  const int64_t groups = (cols + kBlock - 1) / kBlock;
  g.rows = rows;
  g.cols = cols;
  g.groups = (int)groups;
  int64_t taken = groups;
  for (g.across = 16; g.across > 1; g.across /= 2) {
    taken = (groups + g.across - 1) / g.across * g.across;
    if (4 * (taken - groups) <= taken) break;
  }
  if (g.across == 1) taken = groups;
  const int64_t down = (int64_t)(16 / g.across) * kUnroll, blocks = (rows + down - 1) / down;
  grid = dim3((unsigned)(taken / g.across), (unsigned)(blocks < 32768 ? blocks : 32768));
  return groups <= (int64_t)1 << 24;
}

template <typename F>
int by_type(int dtype, F&& f) {
  switch (dtype) {
    case HPFP8_OUT_BF16: f(Bf16()); return HPFP8_OK;
    case HPFP8_OUT_F32: f(F32()); return HPFP8_OK;
    case HPFP8_TYPE_F16: f(F16()); return HPFP8_OK;
  }
  return fail(HPFP8_ERR_ARG, "unknown element type %d", dtype);
}

template <typename F>
void by_kind(int kind, F&& f) {
  switch (kind) {
    case kSilu: f(std::integral_constant<int, kSilu>()); break;
    case kGelu: f(std::integral_constant<int, kGelu>()); break;
    case kGeluTanh: f(std::integral_constant<int, kGeluTanh>()); break;
    default: f(std::integral_constant<int, kSwiglu>());
  }
}

bool at_element(const void* p, int dtype) { return ((uintptr_t)p & (dtype == HPFP8_OUT_F32 ? 3 : 1)) == 0; }

template <bool SPECIAL>
int quantize_rows(const void* x, int dtype, int64_t rows, int64_t cols, int64_t ld, void* q, float* scale_inv, hpfp8_stream_t stream) {
  HPFP8_REQUIRE(dtype >= 0 && dtype <= 2, HPFP8_ERR_ARG, "unknown element type %d", dtype);
  HPFP8_REQUIRE(rows >= 0 && cols >= 0 && ld >= 0, HPFP8_ERR_SHAPE, "negative size (rows=%lld cols=%lld ld=%lld)", (long long)rows, (long long)cols, (long long)ld);
  if (rows == 0 || cols == 0) return HPFP8_OK;
  HPFP8_REQUIRE(x && q && scale_inv, HPFP8_ERR_ARG, "null buffer");
  HPFP8_REQUIRE(at_element(x, dtype), HPFP8_ERR_ALIGN, "x is not aligned to its elements");
  Grid g;
  dim3 grid;
  HPFP8_REQUIRE(shape(rows, cols, g, grid), HPFP8_ERR_SHAPE, "a row of %lld values is too long", (long long)cols);
  const int rc = by_type(dtype, [&](auto e) {
    using E = decltype(e);
    quantize_rows_kernel<E, SPECIAL><<<grid, 256, 0, (hipStream_t)stream>>>((const typename E::raw*)x, ld, g, (uint8_t*)q, scale_inv);
  });
  return rc != HPFP8_OK ? rc : check_launch("quantize_rows");
}

template <bool SPECIAL>
int dequantize_rows(const void* q, const float* scale_inv, int64_t rows, int64_t cols, void* x, int dtype, hpfp8_stream_t stream) {
  HPFP8_REQUIRE(dtype >= 0 && dtype <= 2, HPFP8_ERR_ARG, "unknown element type %d", dtype);
  HPFP8_REQUIRE(rows >= 0 && cols >= 0, HPFP8_ERR_SHAPE, "negative size (rows=%lld cols=%lld)", (long long)rows, (long long)cols);
  if (rows == 0 || cols == 0) return HPFP8_OK;
  HPFP8_REQUIRE(x && q && scale_inv, HPFP8_ERR_ARG, "null buffer");
  HPFP8_REQUIRE(at_element(x, dtype), HPFP8_ERR_ALIGN, "x is not aligned to its elements");
  Grid g;
  dim3 grid;
  HPFP8_REQUIRE(shape(rows, cols, g, grid), HPFP8_ERR_SHAPE, "a row of %lld values is too long", (long long)cols);
  const int rc = by_type(dtype, [&](auto e) {
    using E = decltype(e);
    dequantize_rows_kernel<E, SPECIAL><<<grid, 256, 0, (hipStream_t)stream>>>((const uint8_t*)q, scale_inv, g, (typename E::raw*)x);
  });
  return rc != HPFP8_OK ? rc : check_launch("dequantize_rows");
}

}  // namespace
}  // namespace hpfp8

using namespace hpfp8;

extern "C" {

int hpfp8_quantize_rows(const void* x, int dtype, int64_t rows, int64_t cols, int64_t ld, void* q, float* scale_inv, hpfp8_stream_t stream) {
  return quantize_rows<false>(x, dtype, rows, cols, ld, q, scale_inv, stream);
}
int hpfp8_quantize_saved_rows(const void* x, int dtype, int64_t rows, int64_t cols, int64_t ld, void* q, float* scale_inv, hpfp8_stream_t stream) {
  return quantize_rows<true>(x, dtype, rows, cols, ld, q, scale_inv, stream);
}
int hpfp8_dequantize_rows(const void* q, const float* scale_inv, int64_t rows, int64_t cols, void* x, int dtype, hpfp8_stream_t stream) {
  return dequantize_rows<false>(q, scale_inv, rows, cols, x, dtype, stream);
}
int hpfp8_dequantize_saved_rows(const void* q, const float* scale_inv, int64_t rows, int64_t cols, void* x, int dtype, hpfp8_stream_t stream) {
  return dequantize_rows<true>(q, scale_inv, rows, cols, x, dtype, stream);
}

int hpfp8_activation_forward(const void* x, int dtype, int64_t rows, int64_t cols, int64_t ld, int kind, void* y, void* q, float* scale_inv,
                             hpfp8_stream_t stream) {
  HPFP8_REQUIRE(dtype >= 0 && dtype <= 2, HPFP8_ERR_ARG, "unknown element type %d", dtype);
  HPFP8_REQUIRE(kind >= kSilu && kind <= kSwiglu, HPFP8_ERR_ARG, "unknown activation %d", kind);
  HPFP8_REQUIRE(rows >= 0 && cols >= 0 && ld >= 0, HPFP8_ERR_SHAPE, "negative size (rows=%lld cols=%lld ld=%lld)", (long long)rows, (long long)cols, (long long)ld);
  if (rows == 0 || cols == 0) return HPFP8_OK;
  HPFP8_REQUIRE(x && y && (!q == !scale_inv), HPFP8_ERR_ARG, "null buffer, or codes without scales");
  HPFP8_REQUIRE(at_element(x, dtype) && at_element(y, dtype), HPFP8_ERR_ALIGN, "a tensor is not aligned to its elements");
  Grid g;
  dim3 grid;
  HPFP8_REQUIRE(shape(rows, cols, g, grid), HPFP8_ERR_SHAPE, "a row of %lld values is too long", (long long)cols);
  const int rc = by_type(dtype, [&](auto e) {
    using E = decltype(e);
    using raw = typename E::raw;
    by_kind(kind, [&](auto k) {
      if (q) activation_forward_kernel<E, k, true><<<grid, 256, 0, (hipStream_t)stream>>>((const raw*)x, ld, g, (raw*)y, (uint8_t*)q, scale_inv);
      else activation_forward_kernel<E, k, false><<<grid, 256, 0, (hipStream_t)stream>>>((const raw*)x, ld, g, (raw*)y, nullptr, nullptr);
    });
  });
  return rc != HPFP8_OK ? rc : check_launch("activation_forward");
}

int hpfp8_activation_backward(const void* dy, const void* x, int64_t ld, const void* q, const float* scale_inv, int dtype, int64_t rows,
                              int64_t cols, int kind, void* dx, hpfp8_stream_t stream) {
  HPFP8_REQUIRE(dtype >= 0 && dtype <= 2, HPFP8_ERR_ARG, "unknown element type %d", dtype);
  HPFP8_REQUIRE(kind >= kSilu && kind <= kSwiglu, HPFP8_ERR_ARG, "unknown activation %d", kind);
  HPFP8_REQUIRE(rows >= 0 && cols >= 0 && ld >= 0, HPFP8_ERR_SHAPE, "negative size (rows=%lld cols=%lld ld=%lld)", (long long)rows, (long long)cols, (long long)ld);
  if (rows == 0 || cols == 0) return HPFP8_OK;
  HPFP8_REQUIRE(dy && dx && (!q == !scale_inv) && (!x != !q), HPFP8_ERR_ARG, "null buffer, codes without scales, or not one of x and its codes");
  HPFP8_REQUIRE(at_element(dy, dtype) && at_element(dx, dtype) && at_element(x, dtype), HPFP8_ERR_ALIGN, "a tensor is not aligned to its elements");
  Grid g;
  dim3 grid;
  HPFP8_REQUIRE(shape(rows, cols, g, grid), HPFP8_ERR_SHAPE, "a row of %lld values is too long", (long long)cols);
  const int rc = by_type(dtype, [&](auto e) {
    using E = decltype(e);
    using raw = typename E::raw;
    by_kind(kind, [&](auto k) {
      if (q)
        activation_backward_kernel<E, k, true><<<grid, 256, 0, (hipStream_t)stream>>>((const raw*)dy, nullptr, 0, (const uint8_t*)q, scale_inv, g, (raw*)dx);
      else
        activation_backward_kernel<E, k, false><<<grid, 256, 0, (hipStream_t)stream>>>((const raw*)dy, (const raw*)x, ld, nullptr, nullptr, g, (raw*)dx);
    });
  });
  return rc != HPFP8_OK ? rc : check_launch("activation_backward");
}

}  // extern "C"
