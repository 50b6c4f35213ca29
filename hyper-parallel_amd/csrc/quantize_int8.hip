// Rows of values -> int8 codes with one scale for each row: what hpfp8_gemm_int8 reads.
//
//   v = x[r, c] (times column_scale[c], rounded to fp32),   amax_r = max |v|,   code = rint(v * (127 / amax_r)),   scale_inv_r = amax_r / 127
//
// amax_r is at least 1e-12, as everywhere; with column scales at least 2^-118.  Those rows are a gradient's, which a loss averaged over many tokens
// makes far smaller than 1e-12 before the scales, 1e-3 and less, are on it: all its codes would be 0.
//
// Bound by memory: x is read once, a row in the registers of a team of 16 to 512 threads while its largest value is found, the next row's
// loads under way.  Rows longer than 16384 values are read twice, the second time through the L2.
// bf16: 16384 x 7168 60 us, 5.8 TB/s; 4096 x 16384 36 us, 5.6 TB/s; 2048 x 40960 61 us, 4.1 TB/s; 8 x 7168 2.8 us.
#include "norm_rows.h"

namespace hpfp8 {
namespace {

constexpr int64_t kMaxInt8Cols = 130944;       // (the contraction that a product's 32-bit sums hold, codes of -128 among them)

// the least amax whose two scales are normal numbers: 127 * 2^118 < 2^125, and 2^-118 / 127 > 2^-126
constexpr float kLeastOfColumns = 0x1p-118f;

struct Int8Params {
  const void* x;
  int64_t ld;                   // elements between the rows of x
  int64_t rows;
  int cols;
  const float* column_scale;    // may be null
  uint8_t* q;                   // [rows, cols]
  float* scale_inv;             // [rows]
};

template <typename E, int TPR, int NV, bool COLUMNS>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void quantize_int8_kernel(Int8Params p) {
  using raw = typename E::raw;
  constexpr int kTeams = (TPR < 256 ? 256 : TPR) / TPR, kWaves = TPR < 64 ? 1 : TPR / 64;
  __shared__ float tops[2][kTeams][kWaves];
  const int team = team_of<TPR>(), t = threadIdx.x % TPR, wave = __builtin_amdgcn_readfirstlane(t / 64);
  const int C = p.cols;
  Chunk at[NV];
  float by[COLUMNS ? NV : 1][8];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    at[j] = chunk_at<kWhole>(j * TPR + t, C);
    if constexpr (COLUMNS) load8<F32, false>(p.column_scale + at[j].col, at[j].any ? 8 : 0, by[j]);
  }
  const int64_t step = (int64_t)gridDim.x * kTeams, first = (int64_t)blockIdx.x * kTeams;
  Pack8<E> next[NV];
  auto fetch = [&](int64_t r) {
#pragma unroll
    for (int j = 0; j < NV; ++j) next[j] = load_chunk<E, kWhole>((const raw*)p.x + (r < p.rows ? r : 0) * p.ld, at[j], C, r < p.rows);
  };
  fetch(first + team);
  int turn = 0;
  for (int64_t from = first; from < p.rows; from += step, turn ^= 1) {       // (as many turns for every team)
    const int64_t row = from + team;
    float v[NV][8];
    float top = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) unpack8<E>(next[j], v[j]);
    fetch(row + step);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if constexpr (COLUMNS) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[j][i] *= by[j][i];
      }
      top = __uint_as_float(umax(__float_as_uint(top), __float_as_uint(at[j].any ? magnitude8(v[j]) : 0.f)));
    }
    top = magnitude_over<(TPR >= 64)>(top);
    if constexpr (kWaves > 1) {
      if ((t & 63) == 0) tops[turn][team][wave] = top;
      __syncthreads();                                                        // (the next turn writes the other half)
      uint32_t m = 0;
#pragma unroll
      for (int k = 0; k < kWaves; ++k) m = umax(m, __float_as_uint(tops[turn][team][k]));
      top = __uint_as_float(m);
    }
    if (row >= p.rows) continue;
    float scale, si;
    int8_scales(top, scale, si, COLUMNS ? kLeastOfColumns : kAmaxEps);
    if (t == 0) p.scale_inv[row] = si;
#pragma unroll
    for (int j = 0; j < NV; ++j) store_chunk_codes<kWhole>(p.q + row * C, at[j], C, int8_codes(v[j], scale, top < INFINITY));
  }
}

// One workgroup per row, which it walks through twice.
template <typename E, bool COLUMNS>
__global__ __launch_bounds__(1024) void quantize_int8_long_kernel(Int8Params p) {
  using raw = typename E::raw;
  __shared__ float tops[16];
  const int t = threadIdx.x, wave = t >> 6;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const raw* const x = (const raw*)p.x + row * p.ld;
    auto values = [&](int col, float v[8]) {
      load8<E, false>(x + col, 8, v);
      if constexpr (COLUMNS) {
        float by[8];
        load8<F32, false>(p.column_scale + col, 8, by);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] *= by[i];
      }
    };
    uint32_t m = 0;
    for (int col = t * 8; col < p.cols; col += 1024 * 8) {
      float v[8];
      values(col, v);
      m = umax(m, __float_as_uint(magnitude8(v)));
    }
    const float mine = magnitude_over<true>(__uint_as_float(m));
    if ((t & 63) == 0) tops[wave] = mine;
    __syncthreads();
    m = 0;
#pragma unroll
    for (int k = 0; k < 16; ++k) m = umax(m, __float_as_uint(tops[k]));
    const float top = __uint_as_float(m);
    __syncthreads();                                                          // (the next row writes it again)
    float scale, si;
    int8_scales(top, scale, si, COLUMNS ? kLeastOfColumns : kAmaxEps);
    if (t == 0) p.scale_inv[row] = si;
    for (int col = t * 8; col < p.cols; col += 1024 * 8) {
      float v[8];
      values(col, v);
      store_codes8<false>(p.q + row * p.cols + col, 8, int8_codes(v, scale, top < INFINITY));
    }
  }
}

template <bool COLUMNS>
void launch(const Int8Params& p, int dtype, hipStream_t stream) {
  if (p.cols > kMaxCols) {
    const dim3 grid((unsigned)(p.rows < 1024 ? p.rows : 1024));
    if (dtype == HPFP8_OUT_BF16) quantize_int8_long_kernel<Bf16, COLUMNS><<<grid, 1024, 0, stream>>>(p);
    else if (dtype == HPFP8_TYPE_F16) quantize_int8_long_kernel<F16, COLUMNS><<<grid, 1024, 0, stream>>>(p);
    else quantize_int8_long_kernel<F32, COLUMNS><<<grid, 1024, 0, stream>>>(p);
    return;
  }
  by_type_and_width<false>(dtype, p.cols, [&](auto e, auto tpr, auto nv) {
    constexpr int kThreads = tpr < 256 ? 256 : tpr, kTeams = kThreads / tpr;
    const int64_t blocks = (p.rows + kTeams - 1) / kTeams, most = 256 * (2048 / kThreads);
    quantize_int8_kernel<decltype(e), tpr, nv, COLUMNS><<<dim3((unsigned)(blocks < most ? blocks : most)), kThreads, 0, stream>>>(p);
  });
}

}  // namespace
}  // namespace hpfp8

using namespace hpfp8;

extern "C" int hpfp8_quantize_int8(const void* x, int dtype, int64_t rows, int64_t cols, int64_t ld, const float* column_scale, void* q,
                                   float* scale_inv, hpfp8_stream_t stream) {
  HPFP8_REQUIRE(dtype >= 0 && dtype <= 2, HPFP8_ERR_ARG, "unknown element type %d", dtype);
  HPFP8_REQUIRE(rows >= 0 && cols > 0, HPFP8_ERR_SHAPE, "rows=%lld cols=%lld", (long long)rows, (long long)cols);
  HPFP8_REQUIRE(cols % kBlock == 0 && cols <= kMaxInt8Cols, HPFP8_ERR_SHAPE, "a row of %lld values is not a multiple of %d of at most %lld",
                (long long)cols, kBlock, (long long)kMaxInt8Cols);
  if (rows == 0) return HPFP8_OK;
  HPFP8_REQUIRE(x && q && scale_inv, HPFP8_ERR_ARG, "null buffer");
  HPFP8_REQUIRE(ld >= 0, HPFP8_ERR_SHAPE, "negative stride");
  HPFP8_REQUIRE(at_element(x, dtype) && at_element(column_scale, HPFP8_OUT_F32) && at_element(scale_inv, HPFP8_OUT_F32), HPFP8_ERR_ALIGN,
                "a tensor is not aligned to its elements");
  const Int8Params p = {x, ld, rows, (int)cols, column_scale, (uint8_t*)q, scale_inv};
  if (column_scale) launch<true>(p, dtype, (hipStream_t)stream);
  else launch<false>(p, dtype, (hipStream_t)stream);
  return check_launch("quantize_int8");
}
