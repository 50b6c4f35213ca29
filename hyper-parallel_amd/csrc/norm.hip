// Layer norm over the last dimension, forward and backward, its normalised input kept for the backward in 8 bits if asked for.
//
//   hat = (x - mean(x)) / sqrt(mean((x - mean)^2) + eps),   y = hat w + b
//   u = dy w,   dx = (u - mean(u) - hat mean(u hat)) / sqrt(...),   dw = sum over rows of dy hat,   db = sum over rows of dy
//
// One pass over memory each way, bound by it: a row is in the registers of a team of 16 to 512 threads, eight neighbouring
// values per thread and step, from its load to its results.  All sums are fp32; the variance is taken around the mean (each wave's
// values around the wave's own mean, the waves joined by their counts), so an offset many times the spread costs nothing.
// The workgroups stay for many rows: the weight's values are loaded once, the next row's loads are under way while a row is worked on,
// and in the backward the two vectors' gradients grow in registers.  At the end a workgroup's teams are joined in LDS in their order and
// its sums leave as one row of partial sums, at most 256 of them (512 where rows are short), which a second launch adds up in a fixed
// order: the same bits every time, and for 4096 rows of 7168 14 MB of sums beside 176 MB of values.
//
// bf16: 4096 x 7168 forward 24 us, 4.9 TB/s, backward 36 + 4 us, 4.9 TB/s; 16384 x 7168 kept in 8 bits 114 us, 5.2 TB/s, and 112 + 4; 8 x 7168 4.4 us,
// a launch's latency with one row's.
#include "norm_rows.h"

namespace hpfp8 {
namespace {

constexpr int kMaxPartials = 256;          // one workgroup of the backward per compute unit (two where rows are short)

struct NormParams {
  const void* x;
  int64_t ld;            // elements between the rows of x
  const void* w;         // may be null, as b
  const void* b;
  int wtype;             // element type of w and b: HPFP8_OUT_BF16, HPFP8_OUT_F32 or HPFP8_TYPE_F16
  int64_t rows;
  int cols;
  float eps;
  void* y;
  float* mean;           // [rows], may be null
  float* rstd;           // [rows], may be null
  uint8_t* q;            // [rows, cols] codes of hat
  float* scale_inv;      // [rows, ceil(cols / 128)]
  const void* dy;
  int64_t ld_dy;
  void* dx;
  float* partial;        // [workgroups][2][cols]: dw, db
};

// A row per team of TPR threads; thread t has the chunks of eight values t, t + TPR, ...: 16 neighbouring threads have one group of 128.
template <typename E, int TPR, int NV, bool KEEP, int EDGE>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR, NV <= 2 && sizeof(typename E::raw) == 2 ? 4 : 2) void norm_forward_kernel(NormParams p) {
  using raw = typename E::raw;
  constexpr int kTeams = (TPR < 256 ? 256 : TPR) / TPR, kWaves = TPR < 64 ? 1 : TPR / 64;
  // (four rows on their way where they fit the registers of two workgroups a compute unit: 16384 x 5120 70.6 / 65.9 us, x 7168 90.8 / 87.7, x 8192
  // 93.5 / 91.9; with codes they do not, 118 us with two and 158 with four, nor with the masks of rows that are no multiple of 128)
  constexpr int kAhead = TPR == 512 && NV == 2 && !KEEP && EDGE == kWhole && sizeof(raw) == 2 ? 4 : 2;
  __shared__ v4f parts[2][kTeams][kWaves];
  const int team = team_of<TPR>(), t = threadIdx.x % TPR, wave = __builtin_amdgcn_readfirstlane(t / 64);
  const int C = p.cols, groups = (C + kBlock - 1) / kBlock;
  Chunk at[NV];
  bool live[NV];         // whether this wave has any of the step's values: with none it does nothing (4104 values are one more than a step's)
  bool cut[NV];          // whether some of the step's chunks are not there, or not whole: only then are values looked at one by one
                         // (16384 x 4104 77 us otherwise, 71)
  float w[NV][8], b[NV][8];
  int mine = 0;                                       // values of a row in this wave's hands
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    at[j] = chunk_at<EDGE>(j * TPR + t, C);
    live[j] = j == 0 && TPR <= 64 ? true : (j * TPR + wave * 64) * 8 < C;
    cut[j] = EDGE == kSingle || (j * TPR + (TPR < 64 ? TPR : wave * 64 + 64)) * 8 > C;
    const int left = C - (j * TPR + wave * 64) * 8, most = (TPR < 64 ? TPR : 64) * 8;
    mine += left < 0 ? 0 : (left < most ? left : most);
    vector_chunk<EDGE>(p.w, p.wtype, at[j], C, 1.f, w[j]);
    vector_chunk<EDGE>(p.b, p.wtype, at[j], C, 0.f, b[j]);
  }
  const float n = (float)mine;
  const int64_t step = (int64_t)gridDim.x * kTeams;
  Pack8<E> next[kAhead][NV];
  auto fetch = [&](Pack8<E> (&to)[NV], int64_t r) {
#pragma unroll
    for (int j = 0; j < NV; ++j) to[j] = load_chunk<E, EDGE>((const raw*)p.x + (r < p.rows ? r : 0) * p.ld, at[j], C, r < p.rows);
  };
  auto work = [&](const Pack8<E> (&packed)[NV], int64_t row, int turn) {
    float v[NV][8];
#pragma unroll
    for (int j = 0; j < NV; ++j) unpack8<E>(packed[j], v[j]);
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (live[j]) {
        if (EDGE == kOverlap && cut[j]) {
#pragma unroll
          for (int i = 0; i < 8; ++i) s += i < 7 && i < at[j].dup ? 0.f : v[j][i];
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) s += v[j][i];
        }
      }
    float mean = mine ? team_sum<TPR>(s) / n : 0.f;
    float m2 = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (live[j]) {
        if (cut[j]) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float d = own<EDGE>(at[j], i, C) ? v[j][i] - mean : 0.f;
            m2 = __builtin_fmaf(d, d, m2);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float d = v[j][i] - mean;
            m2 = __builtin_fmaf(d, d, m2);
          }
        }
      }
    m2 = team_sum<TPR>(m2);
    if constexpr (kWaves > 1) {
      if ((t & 63) == 0) parts[turn][team][wave] = v4f{n, mean, m2, 0.f};
      __syncthreads();                                // (one barrier: the next turn writes the other half)
      float total = 0.f;
#pragma unroll
      for (int k = 0; k < kWaves; ++k) total += parts[turn][team][k][0] * parts[turn][team][k][1];
      mean = total / (float)C;
      m2 = 0.f;
#pragma unroll
      for (int k = 0; k < kWaves; ++k) {
        const v4f each = parts[turn][team][k];
        m2 += each[2] + each[0] * ((each[1] - mean) * (each[1] - mean));
      }
    }
    const float rstd = 1.0f / sqrtf(m2 / (float)C + p.eps);
    if (row >= p.rows) return;
    if (t == 0) {
      if (p.mean) p.mean[row] = mean;
      if (p.rstd) p.rstd[row] = rstd;
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (!live[j]) continue;
      float out[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[j][i] = (v[j][i] - mean) * rstd;
        out[i] = __builtin_fmaf(v[j][i], w[j][i], b[j][i]);
      }
      store_chunk<E, EDGE>((raw*)p.y + row * C, at[j], C, out);
      if constexpr (KEEP) {
        float si;
        if (cut[j]) {                                 // (a group's maximum is that of its own values)
#pragma unroll
          for (int i = 0; i < 8; ++i) v[j][i] = own<EDGE>(at[j], i, C) ? v[j][i] : 0.f;
        }
        const uint2 c = encode_group(v[j], si);
        store_chunk_codes<EDGE>(p.q + row * C, at[j], C, c);
        if (at[j].any && (t & 15) == 0) p.scale_inv[row * groups + (j * TPR + t) / 16] = si;
      }
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
      Pack8<E> packed[NV];
#pragma unroll
      for (int j = 0; j < NV; ++j) packed[j] = next[u][j];
      fetch(next[u], from + team + kAhead * step);
      work(packed, from + team, turn);
    }
  }
}

constexpr int kBackwardThreads = 512;
template <typename E, int TPR, int NV, bool KEEP, int EDGE>
__global__ __launch_bounds__(kBackwardThreads) void norm_backward_kernel(NormParams p) {
  using raw = typename E::raw;
  constexpr int kTeams = kBackwardThreads / TPR, kWaves = TPR < 64 ? 1 : TPR / 64, kChunks = TPR * NV;
  // (rows on their way: teams of a wave and less have several anyway, 65536 x 1024 79 us with three and 80 with four; a wider row is in more hands, 16384 x
  // 5120 99 / 95, x 7168 kept in 8 bits 120 / 115; of over 8192 values four steps' sums fill half of the registers: one row, the weight in LDS)
  constexpr int kAhead = NV > 2 ? 1 : (TPR >= 256 && sizeof(raw) == 2 ? 4 : 3);
  constexpr bool kHoldWeight = NV <= 2;
  __shared__ v2f parts[2][kTeams][kWaves];
  __shared__ v4f joined[kTeams > 1 ? 2 * kChunks * 2 : 1];
  __shared__ v4f weight[kHoldWeight ? 1 : kChunks * 2];
  const int team = team_of<TPR>(), t = threadIdx.x % TPR, wave = __builtin_amdgcn_readfirstlane(t / 64);
  const int C = p.cols, groups = (C + kBlock - 1) / kBlock;
  Chunk at[NV];
  bool live[NV];         // whether this wave has any of the step's values: with none it does nothing (4104 values are one more than a step's)
  float w[kHoldWeight ? NV : 1][8], dw[NV][8], db[NV][8];
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
    for (int i = 0; i < 8; ++i) dw[j][i] = db[j][i] = 0.f;
  }
  const int64_t step = (int64_t)gridDim.x * kTeams;
  struct Row {
    Pack8<E> dy[NV], x[KEEP ? 1 : NV];
    uint2 q[KEEP ? NV : 1];
    float s[KEEP ? NV : 1], mean, rstd;
  };
  Row next[kAhead];
  auto fetch = [&](Row& to, int64_t r) {
    const bool in = r < p.rows;
    const int64_t row = in ? r : 0;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      to.dy[j] = load_chunk<E, EDGE>((const raw*)p.dy + row * p.ld_dy, at[j], C, in);
      if constexpr (KEEP) {
        to.q[j] = load_codes8<EDGE == kSingle>(p.q + row * C + at[j].col, in && at[j].any ? (EDGE == kSingle ? C - at[j].col : 8) : 0);
        to.s[j] = in && at[j].any ? (p.scale_inv + row * groups)[(j * TPR + t) / 16] : 0.f;
      } else {
        to.x[j] = load_chunk<E, EDGE>((const raw*)p.x + row * p.ld, at[j], C, in);
      }
    }
    to.mean = !KEEP && in ? p.mean[row] : 0.f;
    to.rstd = in ? p.rstd[row] : 0.f;
  };
  auto work = [&](const Row& from, int64_t row, int turn) {
    float go[NV][8], hat[NV][8];
    const float rstd = from.rstd;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (!live[j]) continue;
      unpack8<E>(from.dy[j], go[j]);
      if constexpr (KEEP) {
        decode8(from.q[j], from.s[j], hat[j]);        // (the values before a chunk's own have another group's scale: they are not used)
      } else {
        unpack8<E>(from.x[j], hat[j]);
#pragma unroll
        for (int i = 0; i < 8; ++i) hat[j][i] = (hat[j][i] - from.mean) * rstd;
      }
    }
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (!live[j]) continue;
      if (!kHoldWeight) {
#pragma unroll
        for (int i = 0; i < 8; ++i) w[0][i] = weight[(j * TPR + t) * 2 + i / 4][i % 4];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        dw[j][i] = __builtin_fmaf(go[j][i], hat[j][i], dw[j][i]);
        db[j][i] += go[j][i];
        go[j][i] *= w[kHoldWeight ? j : 0][i];        // from here on u
        // (where there is nothing, go is 0, and x and mean with it or finite)
        const float u = EDGE == kOverlap && i < 7 && i < at[j].dup ? 0.f : go[j][i];
        s1 += u;
        s2 = EDGE == kOverlap && i < 7 && i < at[j].dup ? s2 : __builtin_fmaf(u, hat[j][i], s2);
      }
    }
    s1 = team_sum<TPR>(s1);
    s2 = team_sum<TPR>(s2);
    if constexpr (kWaves > 1) {
      if ((t & 63) == 0) parts[turn][team][wave] = v2f{s1, s2};
      __syncthreads();
      s1 = s2 = 0.f;
#pragma unroll
      for (int k = 0; k < kWaves; ++k) {
        s1 += parts[turn][team][k].x;
        s2 += parts[turn][team][k].y;
      }
    }
    if (row >= p.rows) return;
    const float m1 = s1 / (float)C, m2 = s2 / (float)C;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (!live[j]) continue;
      float out[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) out[i] = (go[j][i] - m1 - hat[j][i] * m2) * rstd;
      store_chunk<E, EDGE>((raw*)p.dx + row * C, at[j], C, out);
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
  // the teams' sums, one after the other
  float* const to = p.partial + (int64_t)blockIdx.x * 2 * C;
  for (int k = 0; k < kTeams; ++k) {
    if (team == k) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if constexpr (kTeams > 1) {
          v4f* const a = joined + (j * TPR + t) * 2;
          v4f* const b = joined + (kChunks + j * TPR + t) * 2;
          if (k > 0) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              dw[j][i] = a[i / 4][i % 4] + dw[j][i];
              db[j][i] = b[i / 4][i % 4] + db[j][i];
            }
          }
          if (k < kTeams - 1) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              a[h] = v4f{dw[j][4 * h], dw[j][4 * h + 1], dw[j][4 * h + 2], dw[j][4 * h + 3]};
              b[h] = v4f{db[j][4 * h], db[j][4 * h + 1], db[j][4 * h + 2], db[j][4 * h + 3]};
            }
          }
        }
        if (k == kTeams - 1) {
          store_chunk<F32, EDGE>(to, at[j], C, dw[j]);
          store_chunk<F32, EDGE>(to + C, at[j], C, db[j]);
        }
      }
    }
    if (kTeams > 1) __syncthreads();
  }
}

// dw and db from the workgroups' partial sums: 64 columns per workgroup, each of its 16 waves every sixteenth partial sum, then the waves in order.
__global__ __launch_bounds__(1024) void norm_join_kernel(const float* __restrict__ partial, int count, int cols, void* __restrict__ dw,
                                                         void* __restrict__ db, int wtype) {
  __shared__ float parts[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t col = (int64_t)blockIdx.x * 64 + lane, all = 2 * (int64_t)cols;
  float s = 0.f;
  if (col < all) {
    int k = wave;
    for (; k + 48 < count; k += 64) {
      float v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) v[u] = partial[(k + 16 * u) * all + col];
#pragma unroll
      for (int u = 0; u < 4; ++u) s += v[u];
    }
    for (; k < count; k += 16) s += partial[k * all + col];
  }
  parts[wave][lane] = s;
  __syncthreads();
  if (wave == 0 && col < all) {
    float total = 0.f;
#pragma unroll
    for (int k = 0; k < 16; ++k) total += parts[k][lane];
    void* const to = col < cols ? dw : db;
    const int64_t i = col < cols ? col : col - cols;
    if (!to) return;
    if (wtype == HPFP8_OUT_BF16) ((uint16_t*)to)[i] = from_f32<Bf16>(total);
    else if (wtype == HPFP8_TYPE_F16) ((_Float16*)to)[i] = (_Float16)total;
    else ((float*)to)[i] = total;
  }
}

template <int TPR, int NV, typename F>
void by_form(bool keep, int cols, F&& f) {
  auto with = [&](auto edge) {
    if (keep) f(std::true_type(), edge);
    else f(std::false_type(), edge);
  };
  if constexpr (TPR * NV == 16) {
    if (cols < 8) return with(std::integral_constant<int, kSingle>());
  }
  if (cols % kBlock == 0) with(std::integral_constant<int, kWhole>());
  else with(std::integral_constant<int, kOverlap>());
}

int backward_teams(int64_t cols) {
  const int64_t chunks = (cols + 7) / 8;
  return chunks <= 32 ? 32 : (chunks <= 128 ? 8 : (chunks <= 512 ? 2 : 1));
}


int check(int dtype, int wtype, int64_t rows, int64_t cols) {
  HPFP8_REQUIRE(dtype >= 0 && dtype <= 2 && wtype >= 0 && wtype <= 2, HPFP8_ERR_ARG, "unknown element type (%d, weight %d)", dtype, wtype);
  HPFP8_REQUIRE(rows >= 0 && cols > 0, HPFP8_ERR_SHAPE, "rows=%lld cols=%lld", (long long)rows, (long long)cols);
  HPFP8_REQUIRE(cols <= kMaxCols, HPFP8_ERR_SHAPE, "a row of %lld values is longer than %d", (long long)cols, kMaxCols);
  return HPFP8_OK;
}

}  // namespace
}  // namespace hpfp8

using namespace hpfp8;

extern "C" {

int64_t hpfp8_layer_norm_partials(int64_t rows, int64_t cols) {
  if (rows <= 0 || cols <= 0 || cols > kMaxCols) return 0;
  const int64_t teams = backward_teams(cols), blocks = (rows + teams - 1) / teams, most = cols <= 2048 ? 2 * kMaxPartials : kMaxPartials;
  return blocks < most ? blocks : most;
}

int hpfp8_layer_norm_forward(const void* x, int dtype, int64_t rows, int64_t cols, int64_t ld, const void* w, const void* b, int wtype, float eps,
                             void* y, float* mean, float* rstd, void* q, float* scale_inv, hpfp8_stream_t stream) {
  const int bad = check(dtype, wtype, rows, cols);
  if (bad != HPFP8_OK) return bad;
  if (rows == 0) return HPFP8_OK;
  HPFP8_REQUIRE(x && y && (!q == !scale_inv), HPFP8_ERR_ARG, "null buffer, or codes without scales");
  HPFP8_REQUIRE(ld >= 0, HPFP8_ERR_SHAPE, "negative stride");
  HPFP8_REQUIRE(at_element(x, dtype) && at_element(y, dtype) && at_element(w, wtype) && at_element(b, wtype), HPFP8_ERR_ALIGN,
                "a tensor is not aligned to its elements");
  NormParams p = {};
  p.x = x;
  p.ld = ld;
  p.w = w;
  p.b = b;
  p.wtype = wtype;
  p.rows = rows;
  p.cols = (int)cols;
  p.eps = eps;
  p.y = y;
  p.mean = mean;
  p.rstd = rstd;
  p.q = (uint8_t*)q;
  p.scale_inv = scale_inv;
  by_type_and_width<false>(dtype, (int)cols, [&](auto e, auto tpr, auto nv) {
    using E = decltype(e);
    constexpr int kThreads = tpr < 256 ? 256 : tpr, kTeams = kThreads / tpr;
    const int64_t blocks = (rows + kTeams - 1) / kTeams, most = 256 * (1024 / kThreads);   // every compute unit full once
    const dim3 grid((unsigned)(blocks < most ? blocks : most));
    by_form<tpr, nv>(q != nullptr, (int)cols,
                     [&](auto keep, auto edge) { norm_forward_kernel<E, tpr, nv, keep, edge><<<grid, kThreads, 0, (hipStream_t)stream>>>(p); });
  });
  return check_launch("layer_norm_forward");
}

int hpfp8_layer_norm_backward(const void* dy, int64_t ld_dy, const void* x, int64_t ld, const float* mean, const void* q, const float* scale_inv,
                              const float* rstd, int dtype, int64_t rows, int64_t cols, const void* w, int wtype, void* dx, void* dw, void* db,
                              float* partial, hpfp8_stream_t stream) {
  const int bad = check(dtype, wtype, rows, cols);
  if (bad != HPFP8_OK) return bad;
  if (rows > 0) {
    HPFP8_REQUIRE(dy && dx && rstd && partial && (!q == !scale_inv) && (q || (x && mean)), HPFP8_ERR_ARG,
                  "null buffer, codes without scales, or neither codes nor x and its mean");
    HPFP8_REQUIRE(ld >= 0 && ld_dy >= 0, HPFP8_ERR_SHAPE, "negative stride");
    HPFP8_REQUIRE(at_element(dy, dtype) && at_element(x, dtype) && at_element(dx, dtype) && at_element(w, wtype) && at_element(dw, wtype) &&
                      at_element(db, wtype), HPFP8_ERR_ALIGN, "a tensor is not aligned to its elements");
    NormParams p = {};
    p.x = x;
    p.ld = ld;
    p.w = w;
    p.wtype = wtype;
    p.rows = rows;
    p.cols = (int)cols;
    p.mean = const_cast<float*>(mean);
    p.rstd = const_cast<float*>(rstd);
    p.q = (uint8_t*)const_cast<void*>(q);
    p.scale_inv = const_cast<float*>(scale_inv);
    p.dy = dy;
    p.ld_dy = ld_dy;
    p.dx = dx;
    p.partial = partial;
    const dim3 grid((unsigned)hpfp8_layer_norm_partials(rows, cols));
    by_type_and_width<true>(dtype, (int)cols, [&](auto e, auto tpr, auto nv) {
      using E = decltype(e);
      by_form<tpr, nv>(q != nullptr, (int)cols, [&](auto keep, auto edge) {
        norm_backward_kernel<E, tpr, nv, keep, edge><<<grid, kBackwardThreads, 0, (hipStream_t)stream>>>(p);
      });
    });
    const int rc = check_launch("layer_norm_backward");
    if (rc != HPFP8_OK) return rc;
  }
  if (dw || db) {      // (no rows: zeros)
    norm_join_kernel<<<(unsigned)((2 * cols + 63) / 64), 1024, 0, (hipStream_t)stream>>>(partial, (int)hpfp8_layer_norm_partials(rows, cols), (int)cols,
                                                                                      dw, db, wtype);
    return check_launch("layer_norm_backward (join)");
  }
  return HPFP8_OK;
}

}  // extern "C"
