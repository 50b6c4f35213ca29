// Backward of the root-mean-square norm:
//
//   hat = s r,   u = dy w,   ds = r (u - hat mean(u hat)) + ds',   dw = sum over rows of dy hat
//
// s: what was normalised (with a residual the sum, whose own gradient ds' is added here: ds is the gradient of x and of the residual).
// One pass over memory like the forward.  The workgroups stay for many rows and dw grows in their registers; at the end a workgroup's teams
// are joined in LDS in their order, its sums leave as one row of partial sums, at most 256 of them (512 where rows are short), and a second
// launch adds those up in a fixed order: the same bits every time.
//
// bf16: 4096 x 7168 with ds' 44 + 4 us, 5.3 TB/s; 16384 x 7168 161 us with both launches, 5.8 TB/s, without ds' 124, 5.7 TB/s.
#include "norm_rows.h"

namespace hpfp8 {
namespace {

constexpr int kMaxPartials = 256;          // one workgroup per compute unit (two where rows are short)
constexpr int kThreads = 512;

struct RmsBackwardParams {
  const void* dy;
  int64_t ld_dy;         // elements between the rows of dy, as the others
  const void* s;
  int64_t ld;
  const void* ds_in;     // may be null
  int64_t ld_ds;
  const float* rstd;     // [rows]
  const void* w;         // may be null
  int wtype;
  int64_t rows;
  int cols;
  void* ds;              // [rows, cols]
  float* partial;        // [workgroups][cols]
};

template <typename E, int TPR, int NV, bool DS, int EDGE>
__global__ __launch_bounds__(kThreads) void rms_backward_kernel(RmsBackwardParams p) {
  using raw = typename E::raw;
  constexpr int kTeams = kThreads / TPR, kWaves = TPR < 64 ? 1 : TPR / 64, kChunks = TPR * NV;
  // Rows on their way while one is worked on, us with two / three / four, with ds': 16384 x 7168 bf16 166 / 163 / 162, x 2048 52 / 55 / 55, 65536 x 256
  // 41 / 44 / 44; 4096 x 16384 with one / two 89 / 80 without ds', with it two do not fit the registers.
  constexpr int kAhead = sizeof(raw) == 4 ? (NV > 2 ? 1 : 2) : (NV > 2 ? (DS ? 1 : 2) : (TPR == 512 ? 4 : (TPR == 256 && NV == 2 ? 3 : 2)));
  constexpr bool kEarlyDs = DS && (NV <= 2 || sizeof(raw) == 2);         // (of over 8192 fp32 values the third stream does not fit the registers)
  constexpr bool kHoldWeight = NV <= 2;      // (four steps' sums and rows fill the registers: the weight in LDS then)
  __shared__ float parts[2][kTeams][kWaves];
  __shared__ v4f joined[kTeams > 1 ? kChunks * 2 : 1];
  __shared__ v4f weight[kHoldWeight ? 1 : kChunks * 2];
  const int team = team_of<TPR>(), t = threadIdx.x % TPR, wave = __builtin_amdgcn_readfirstlane(t / 64);
  const int C = p.cols;
  Chunk at[NV];
  bool live[NV];         // whether this wave has any of the step's values
  float w[kHoldWeight ? NV : 1][8], dw[NV][8];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    at[j] = chunk_at<EDGE>(j * TPR + t, C);
    live[j] = j == 0 && TPR <= 64 ? true : (j * TPR + wave * 64) * 8 < C;
    vector_chunk<EDGE>(p.w, p.wtype, at[j], C, 1.f, w[kHoldWeight ? j : 0]);
    if (!kHoldWeight) {                                // (read by the thread that wrote it)
      weight[(j * TPR + t) * 2] = v4f{w[0][0], w[0][1], w[0][2], w[0][3]};
      weight[(j * TPR + t) * 2 + 1] = v4f{w[0][4], w[0][5], w[0][6], w[0][7]};
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) dw[j][i] = 0.f;
  }
  const int64_t step = (int64_t)gridDim.x * kTeams;
  struct Row {
    Pack8<E> dy[NV], s[NV], ds[kEarlyDs ? NV : 1];
    float rstd;
  };
  Row next[kAhead];
  auto fetch = [&](Row& to, int64_t r) {
    const bool in = r < p.rows;
    const int64_t row = in ? r : 0;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      to.dy[j] = load_chunk<E, EDGE>((const raw*)p.dy + row * p.ld_dy, at[j], C, in);
      to.s[j] = load_chunk<E, EDGE>((const raw*)p.s + row * p.ld, at[j], C, in);
      if constexpr (kEarlyDs) to.ds[j] = load_chunk<E, EDGE>((const raw*)p.ds_in + row * p.ld_ds, at[j], C, in);
    }
    to.rstd = in ? p.rstd[row] : 0.f;
  };
  auto work = [&](const Row& from, int64_t row, int turn) {
    float u[NV][8], hat[NV][8];
    const float rstd = from.rstd;
    float m = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (!live[j]) continue;
      unpack8<E>(from.dy[j], u[j]);
      unpack8<E>(from.s[j], hat[j]);
      if (!kHoldWeight) {
#pragma unroll
        for (int i = 0; i < 8; ++i) w[0][i] = weight[(j * TPR + t) * 2 + i / 4][i % 4];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        hat[j][i] *= rstd;
        dw[j][i] = __builtin_fmaf(u[j][i], hat[j][i], dw[j][i]);
        u[j][i] *= w[kHoldWeight ? j : 0][i];
        m = EDGE == kOverlap && i < 7 && i < at[j].dup ? m : __builtin_fmaf(u[j][i], hat[j][i], m);
      }
    }
    m = team_sum<TPR>(m);
    if constexpr (kWaves > 1) {
      if ((t & 63) == 0) parts[turn][team][wave] = m;
      __syncthreads();                                // (the next turn writes the other half)
      m = 0.f;
#pragma unroll
      for (int k = 0; k < kWaves; ++k) m += parts[turn][team][k];
    }
    if (row >= p.rows) return;
    m /= (float)C;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (!live[j]) continue;
      float out[8], other[8];
      if constexpr (kEarlyDs) unpack8<E>(from.ds[j], other);
      else if constexpr (DS) unpack8<E>(load_chunk<E, EDGE>((const raw*)p.ds_in + row * p.ld_ds, at[j], C, true), other);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        out[i] = (u[j][i] - hat[j][i] * m) * rstd;
        if constexpr (DS) out[i] += other[i];
      }
      store_chunk<E, EDGE>((raw*)p.ds + row * C, at[j], C, out);
    }
  };
  const int64_t first = (int64_t)blockIdx.x * kTeams;
#pragma unroll
  for (int u = 0; u < kAhead; ++u) fetch(next[u], first + team + u * step);
  int turn = 0;
  for (int64_t at_row = first; at_row < p.rows; at_row += kAhead * step) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u, turn ^= 1) {
      const int64_t from = at_row + u * step;         // (as many turns for every team)
      if (from >= p.rows) break;
      const Row row = next[u];
      fetch(next[u], from + team + kAhead * step);
      work(row, from + team, turn);
    }
  }
  // the teams' sums: a wave's four first, then one after the other
  constexpr int kJoint = TPR < 64 ? 4 : 1;
  if constexpr (kJoint > 1) {
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        dw[j][i] += __shfl_xor(dw[j][i], 16);
        dw[j][i] += __shfl_xor(dw[j][i], 32);
      }
  }
  float* const to = p.partial + (int64_t)blockIdx.x * C;
  for (int k = 0; k < kTeams; k += kJoint) {
    if (team == k) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if constexpr (kTeams > 1) {
          v4f* const a = joined + (j * TPR + t) * 2;
          if (k > 0) {
#pragma unroll
            for (int i = 0; i < 8; ++i) dw[j][i] = a[i / 4][i % 4] + dw[j][i];
          }
          if (k < kTeams - kJoint) {
#pragma unroll
            for (int h = 0; h < 2; ++h) a[h] = v4f{dw[j][4 * h], dw[j][4 * h + 1], dw[j][4 * h + 2], dw[j][4 * h + 3]};
          }
        }
        if (k == kTeams - kJoint) store_chunk<F32, EDGE>(to, at[j], C, dw[j]);
      }
    }
    if (kTeams > 1) __syncthreads();
  }
}

// dw from the workgroups' partial sums: 32 columns per workgroup, each of its 32 half waves every 32nd partial sum, then those in order.
__global__ __launch_bounds__(1024) void rms_join_kernel(const float* __restrict__ partial, int count, int cols, void* __restrict__ dw, int wtype) {
  __shared__ float parts[32][33];
  const int lane = threadIdx.x & 31, part = threadIdx.x >> 5;
  const int64_t col = (int64_t)blockIdx.x * 32 + lane;
  float s = 0.f;
  if (col < cols) {
    int k = part;
    for (; k + 224 < count; k += 256) {
      float v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) v[u] = partial[(int64_t)(k + 32 * u) * cols + col];
#pragma unroll
      for (int u = 0; u < 8; ++u) s += v[u];
    }
    for (; k < count; k += 32) s += partial[(int64_t)k * cols + col];
  }
  parts[part][lane] = s;
  __syncthreads();
  if (part == 0 && col < cols) {
    float total = 0.f;
#pragma unroll
    for (int k = 0; k < 32; ++k) total += parts[k][lane];
    if (wtype == HPFP8_OUT_BF16) ((uint16_t*)dw)[col] = from_f32<Bf16>(total);
    else if (wtype == HPFP8_TYPE_F16) ((_Float16*)dw)[col] = (_Float16)total;
    else ((float*)dw)[col] = total;
  }
}

int64_t backward_teams(int64_t cols) {
  const int64_t chunks = (cols + 7) / 8;
  return chunks <= 32 ? 32 : (chunks <= 128 ? 8 : (chunks <= 512 ? 2 : 1));
}

}  // namespace
}  // namespace hpfp8

using namespace hpfp8;

extern "C" {

int64_t hpfp8_rms_norm_partials(int64_t rows, int64_t cols) {
  if (rows <= 0 || cols <= 0 || cols > kMaxCols) return 0;
  const int64_t teams = backward_teams(cols), blocks = (rows + teams - 1) / teams, most = cols <= 2048 ? 2 * kMaxPartials : kMaxPartials;
  return blocks < most ? blocks : most;
}

int hpfp8_rms_norm_backward(const void* dy, int64_t ld_dy, const void* s, int64_t ld, const void* ds_in, int64_t ld_ds, const float* rstd, int dtype,
                            int64_t rows, int64_t cols, const void* w, int wtype, void* ds, void* dw, float* partial, hpfp8_stream_t stream) {
  HPFP8_REQUIRE(dtype >= 0 && dtype <= 2 && wtype >= 0 && wtype <= 2, HPFP8_ERR_ARG, "unknown element type (%d, weight %d)", dtype, wtype);
  HPFP8_REQUIRE(rows >= 0 && cols > 0, HPFP8_ERR_SHAPE, "rows=%lld cols=%lld", (long long)rows, (long long)cols);
  HPFP8_REQUIRE(cols <= kMaxCols, HPFP8_ERR_SHAPE, "a row of %lld values is longer than %d", (long long)cols, kMaxCols);
  HPFP8_REQUIRE(at_element(dw, wtype), HPFP8_ERR_ALIGN, "a tensor is not aligned to its elements");
  if (rows > 0) {
    HPFP8_REQUIRE(dy && s && rstd && ds && partial, HPFP8_ERR_ARG, "null buffer");
    HPFP8_REQUIRE(ld >= 0 && ld_dy >= 0 && ld_ds >= 0, HPFP8_ERR_SHAPE, "negative stride");
    HPFP8_REQUIRE(at_element(dy, dtype) && at_element(s, dtype) && at_element(ds_in, dtype) && at_element(ds, dtype) && at_element(w, wtype),
                  HPFP8_ERR_ALIGN, "a tensor is not aligned to its elements");
    const RmsBackwardParams p = {dy, ld_dy, s, ld, ds_in, ld_ds, rstd, w, wtype, rows, (int)cols, ds, partial};
    const dim3 grid((unsigned)hpfp8_rms_norm_partials(rows, cols));
    by_type_and_width<true>(dtype, (int)cols, [&](auto e, auto tpr, auto nv) {
      using E = decltype(e);
      static_assert(kThreads % tpr == 0, "whole teams");
      auto with = [&](auto edge) {
        if (ds_in) rms_backward_kernel<E, tpr, nv, true, edge><<<grid, kThreads, 0, (hipStream_t)stream>>>(p);
        else rms_backward_kernel<E, tpr, nv, false, edge><<<grid, kThreads, 0, (hipStream_t)stream>>>(p);
      };
      if constexpr (tpr * nv == 16) {
        if (cols < 8) return with(std::integral_constant<int, kSingle>());
      }
      if (cols % kBlock == 0) with(std::integral_constant<int, kWhole>());
      else with(std::integral_constant<int, kOverlap>());
    });
    const int rc = check_launch("rms_norm_backward");
    if (rc != HPFP8_OK) return rc;
  }
  if (dw) {            // (no rows: zeros)
    rms_join_kernel<<<(unsigned)((cols + 31) / 32), 1024, 0, (hipStream_t)stream>>>(partial, (int)hpfp8_rms_norm_partials(rows, cols), (int)cols, dw, wtype);
    return check_launch("rms_norm_backward (join)");
  }
  return HPFP8_OK;
}

}  // extern "C"
