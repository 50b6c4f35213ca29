// Root-mean-square norm over the last dimension, with the addition of a residual ahead of it if asked for.
//
//   s = x + residual (rounded to their type),   y = s r w,   r = 1 / sqrt(mean(s^2) + eps)
//
// One pass over memory: a row is in the registers of a team of 16 to 512 threads, eight neighbouring values per thread and step, from its
// loads to its results, the next row's loads under way.  Sums are fp32.  The result leaves in its own type, or in the 8 bits that the next
// product reads, which are made from its fp32 values: E4M3 with a scale for each 128 of a row (16 threads have such a group), or int8 with
// one for the row (whose largest value is the team's second meeting).
//
// bf16 with the residual: 4096 x 7168 own type 42 us, 5.6 TB/s, E4M3 39 us, 5.4 TB/s, int8 36 us, 5.7 TB/s; 16384 x 7168 154, 141 and 134 us, 6.1, 5.9
// and 6.2 TB/s; without it 79, 76 and 66 us, 5.9, 4.7 and 5.4 TB/s; 8 x 7168 4.5 us, a launch's latency with one row's.
#include "norm_rows.h"

namespace hpfp8 {
namespace {

enum RmsOut { kOwnType, kE4m3, kInt8 };

struct RmsParams {
  const void* x;
  int64_t ld;            // elements between the rows of x
  const void* residual;  // may be null
  int64_t ld_residual;
  const void* w;         // may be null
  int wtype;             // its element type: HPFP8_OUT_BF16, HPFP8_OUT_F32 or HPFP8_TYPE_F16
  int64_t rows;
  int cols;
  float eps;
  void* sum;             // [rows, cols] where there is a residual
  void* y;               // [rows, cols], or codes
  float* rstd;           // [rows], may be null (own type)
  float* scale_inv;      // codes: [cols / 128, rows], or [rows]
  int pow2;              // E4M3: scales that are powers of two
};

// Rows on their way while one is worked on.  us with two / one, 16384 x 7168 bf16, 4096 x 16384: own type 78.5 / 87, 49.1 / 46.7; E4M3 75.2 / 76.8,
// 50.5 / 45.1; int8 70.1 / 65.2, 44.8 / 35.1.  With a residual a row is two streams and (launch_forward) a workgroup has mostly one.
constexpr int rows_ahead(int out, bool residual, int steps) { return residual || steps > 2 || out == kInt8 ? 1 : 2; }

template <typename E, int TPR, int NV, int OUT, bool RES, int EDGE>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR, NV <= 2 && sizeof(typename E::raw) == 2 ? 4 : 2) void rms_forward_kernel(RmsParams p) {
  using raw = typename E::raw;
  constexpr int kTeams = (TPR < 256 ? 256 : TPR) / TPR, kWaves = TPR < 64 ? 1 : TPR / 64;
  constexpr int kAhead = rows_ahead(OUT, RES, NV);
  static_assert(OUT == kOwnType || EDGE == kWhole, "codes are of whole groups");
  __shared__ float sums[2][kTeams][kWaves], tops[2][kTeams][kWaves];
  const int team = team_of<TPR>(), t = threadIdx.x % TPR, wave = __builtin_amdgcn_readfirstlane(t / 64);
  const int C = p.cols;
  Chunk at[NV];
  bool live[NV];         // whether this wave has any of the step's values
  bool cut[NV];          // whether some of the step's chunks are not there, or not whole
  float w[NV][8];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    at[j] = chunk_at<EDGE>(j * TPR + t, C);
    live[j] = j == 0 && TPR <= 64 ? true : (j * TPR + wave * 64) * 8 < C;
    cut[j] = EDGE == kSingle || (j * TPR + (TPR < 64 ? TPR : wave * 64 + 64)) * 8 > C;
    vector_chunk<EDGE>(p.w, p.wtype, at[j], C, 1.f, w[j]);
  }
  struct Row {
    Pack8<E> x[NV], residual[RES ? NV : 1];
  };
  Row next[kAhead];
  auto fetch = [&](Row& to, int64_t r, int64_t end) {
    const bool in = r < end;
    const int64_t row = in ? r : 0;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      to.x[j] = load_chunk<E, EDGE>((const raw*)p.x + row * p.ld, at[j], C, in);
      if constexpr (RES) to.residual[j] = load_chunk<E, EDGE>((const raw*)p.residual + row * p.ld_residual, at[j], C, in);
    }
  };
  auto work = [&](const Row& from, int64_t row, int64_t end, int turn) {
    const bool in = row < end;
    float v[NV][8];
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (!live[j]) continue;
      unpack8<E>(from.x[j], v[j]);
      if constexpr (RES) {
        float other[8];
        unpack8<E>(from.residual[j], other);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[j][i] += other[i];
        if (in) store_chunk<E, EDGE>((raw*)p.sum + row * C, at[j], C, v[j]);
        unpack8<E>(pack8<E>(v[j]), v[j]);             // (the norm is that of the sum as it is stored)
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float d = EDGE == kOverlap && cut[j] && i < 7 && i < at[j].dup ? 0.f : v[j][i];
        ss = __builtin_fmaf(d, d, ss);
      }
    }
    ss = team_sum<TPR>(ss);
    if constexpr (kWaves > 1) {
      if ((t & 63) == 0) sums[turn][team][wave] = ss;
      __syncthreads();                                // (the next turn writes the other half)
      ss = 0.f;
#pragma unroll
      for (int k = 0; k < kWaves; ++k) ss += sums[turn][team][k];
    }
    const float rstd = 1.0f / sqrtf(ss / (float)C + p.eps);
    if (OUT == kOwnType && in && t == 0 && p.rstd) p.rstd[row] = rstd;
    float top = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (!live[j]) continue;
#pragma unroll
      for (int i = 0; i < 8; ++i) v[j][i] = v[j][i] * rstd * w[j][i];
      if constexpr (OUT == kOwnType) {
        if (in) store_chunk<E, EDGE>((raw*)p.y + row * C, at[j], C, v[j]);
      } else if constexpr (OUT == kE4m3) {
        float si;
        const uint2 c = encode_group(v[j], si, p.pow2);
        if (in) store_chunk_codes<EDGE>((uint8_t*)p.y + row * C, at[j], C, c);
        if (in && at[j].any && (t & 15) == 0) p.scale_inv[(int64_t)((j * TPR + t) / 16) * p.rows + row] = si;
      } else {
        // (values that are not there are 0 times rstd times 1: NaN where the row's are)
        const float m = at[j].any ? magnitude8(v[j]) : 0.f;
        top = __uint_as_float(umax(__float_as_uint(top), __float_as_uint(m)));
      }
    }
    if constexpr (OUT == kInt8) {
      top = magnitude_over<(TPR >= 64)>(top);
      if constexpr (kWaves > 1) {
        if ((t & 63) == 0) tops[turn][team][wave] = top;
        __syncthreads();
        uint32_t m = 0;
#pragma unroll
        for (int k = 0; k < kWaves; ++k) m = umax(m, __float_as_uint(tops[turn][team][k]));
        top = __uint_as_float(m);
      }
      float scale, si;
      int8_scales(top, scale, si);
      if (!in) return;
      if (t == 0) p.scale_inv[row] = si;
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (live[j]) store_chunk_codes<EDGE>((uint8_t*)p.y + row * C, at[j], C, int8_codes(v[j], scale, top < INFINITY));
    }
  };
  // E4M3: neighbouring rows are one workgroup's, so that their scales, which lie side by side, meet in one L2.  Otherwise they are spread.
  const int64_t per = (p.rows + (int64_t)gridDim.x * kTeams - 1) / ((int64_t)gridDim.x * kTeams) * kTeams;
  const int64_t first = OUT == kE4m3 ? blockIdx.x * per : (int64_t)blockIdx.x * kTeams;
  const int64_t step = OUT == kE4m3 ? kTeams : (int64_t)gridDim.x * kTeams;
  const int64_t end = OUT == kE4m3 && first + per < p.rows ? first + per : p.rows;
#pragma unroll
  for (int u = 0; u < kAhead; ++u) fetch(next[u], first + team + u * step, end);
  int turn = 0;
  for (int64_t at_row = first; at_row < end; at_row += kAhead * step) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u, turn ^= 1) {
      const int64_t from = at_row + u * step;         // (as many turns for every team)
      if (from >= end) break;
      const Row row = next[u];
      fetch(next[u], from + team + kAhead * step, end);
      work(row, from + team, end, turn);
    }
  }
}

template <int OUT>
int launch_forward(const RmsParams& p, int dtype, hipStream_t stream) {
  by_type_and_width<false>(dtype, p.cols, [&](auto e, auto tpr, auto nv) {
    using E = decltype(e);
    constexpr int kThreads = tpr < 256 ? 256 : tpr, kTeams = kThreads / tpr;
    const int64_t blocks = (p.rows + kTeams - 1) / kTeams, full = 256 * (1024 / kThreads);   // every compute unit full once
    // Workgroups that stay for many rows load the weight once; with a residual, and so two streams written beside two read, ones that leave after
    // one row sweep memory in a tighter order, which is worth more from a few rounds on.  us, staying / leaving, own type, E4M3, int8:
    //   16384 x 7168 bf16  162 / 154, 164 / 141, 147 / 133      65536 x 256  26.2 / 24.3, 24.6 / 22.7, 23.5 / 21.8      fp32 4096 x 7168  92 / 86, 80 / 72, 72 / 69
    //   1024 x 7168        12.1 / 14.1, 13.6 / 13.3, 12.8 / 12.6     4096 x 16384  97 / 90, 94 / 100, 81 / 79;   without a residual 78 / 80, 75 / 79, 65 / 67
    const bool leave = p.residual && blocks > 2 * full && !(OUT == kE4m3 && nv > 2) && blocks < ((int64_t)1 << 22);
    const dim3 grid((unsigned)(leave || blocks < full ? blocks : full));
    auto with = [&](auto edge) {
      if (p.residual) rms_forward_kernel<E, tpr, nv, OUT, true, edge><<<grid, kThreads, 0, stream>>>(p);
      else rms_forward_kernel<E, tpr, nv, OUT, false, edge><<<grid, kThreads, 0, stream>>>(p);
    };
    if constexpr (OUT == kOwnType) {
      if constexpr (tpr * nv == 16) {
        if (p.cols < 8) return with(std::integral_constant<int, kSingle>());
      }
      if (p.cols % kBlock != 0) return with(std::integral_constant<int, kOverlap>());
    }
    with(std::integral_constant<int, kWhole>());
  });
  return check_launch("rms_norm");
}

int check(const RmsParams& p, int dtype, int64_t cols, bool codes) {
  HPFP8_REQUIRE(dtype >= 0 && dtype <= 2 && p.wtype >= 0 && p.wtype <= 2, HPFP8_ERR_ARG, "unknown element type (%d, weight %d)", dtype, p.wtype);
  HPFP8_REQUIRE(p.rows >= 0 && cols > 0, HPFP8_ERR_SHAPE, "rows=%lld cols=%lld", (long long)p.rows, (long long)cols);
  HPFP8_REQUIRE(cols <= kMaxCols, HPFP8_ERR_SHAPE, "a row of %lld values is longer than %d", (long long)cols, kMaxCols);
  HPFP8_REQUIRE(!codes || cols % kBlock == 0, HPFP8_ERR_SHAPE, "a row of %lld values is not a multiple of %d", (long long)cols, kBlock);
  if (p.rows == 0) return HPFP8_OK;
  HPFP8_REQUIRE(p.x && p.y && !p.residual == !p.sum && (!codes || p.scale_inv), HPFP8_ERR_ARG,
                "null buffer, a residual without a sum, or codes without scales");
  HPFP8_REQUIRE(p.ld >= 0 && p.ld_residual >= 0, HPFP8_ERR_SHAPE, "negative stride");
  HPFP8_REQUIRE(at_element(p.x, dtype) && at_element(p.residual, dtype) && at_element(p.sum, dtype) && at_element(p.w, p.wtype) &&
                    (codes || at_element(p.y, dtype)), HPFP8_ERR_ALIGN, "a tensor is not aligned to its elements");
  return 1;
}

}  // namespace
}  // namespace hpfp8

using namespace hpfp8;

extern "C" {

int hpfp8_rms_norm_forward(const void* x, int64_t ld, const void* residual, int64_t ld_residual, int dtype, int64_t rows, int64_t cols, const void* w,
                           int wtype, float eps, void* sum, void* y, float* rstd, hpfp8_stream_t stream) {
  const RmsParams p = {x, ld, residual, ld_residual, w, wtype, rows, (int)cols, eps, sum, y, rstd, nullptr, 0};
  const int rc = check(p, dtype, cols, false);
  return rc <= 0 ? rc : launch_forward<kOwnType>(p, dtype, (hipStream_t)stream);
}

int hpfp8_rms_norm_quantize_1x128_kmajor(const void* x, int64_t ld, const void* residual, int64_t ld_residual, int dtype, int64_t rows, int64_t cols,
                                         const void* w, int wtype, float eps, int pow2, void* sum, void* q, float* scale_inv,
                                         hpfp8_stream_t stream) {
  const RmsParams p = {x, ld, residual, ld_residual, w, wtype, rows, (int)cols, eps, sum, q, nullptr, scale_inv, pow2 != 0};
  const int rc = check(p, dtype, cols, true);
  return rc <= 0 ? rc : launch_forward<kE4m3>(p, dtype, (hipStream_t)stream);
}

int hpfp8_rms_norm_quantize_int8(const void* x, int64_t ld, const void* residual, int64_t ld_residual, int dtype, int64_t rows, int64_t cols,
                                 const void* w, int wtype, float eps, void* sum, void* q, float* scale_inv, hpfp8_stream_t stream) {
  const RmsParams p = {x, ld, residual, ld_residual, w, wtype, rows, (int)cols, eps, sum, q, nullptr, scale_inv, 0};
  const int rc = check(p, dtype, cols, true);
  return rc <= 0 ? rc : launch_forward<kInt8>(p, dtype, (hipStream_t)stream);
}

}  // extern "C"
