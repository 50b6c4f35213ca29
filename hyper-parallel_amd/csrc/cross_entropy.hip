// Softmax cross entropy of a linear's output over a large vocabulary, with its gradients, in pieces of the vocabulary: the logits
// l = x W^T [tokens, vocab] exist as accumulators only.
//
//   lse = log sum_v exp(l_v),  loss = lse - (1 - s) l_target - s mean_v(l_v)                 (s: label smoothing)
//   dl  = c (exp(l - lse) - s / V - (1 - s) [v = target]),  dx = dl W,  dW = dl^T x          (c: the row's share of the loss's gradient)
//
// Forward: one product whose tiles leave, for each row and their columns, the largest logit and the sum of exp(l - largest) in fp32; a second
// launch joins them.  Backward, a piece of the vocabulary at a time: the same product again, whose tiles leave dl rounded to bf16 (at most
// 2^-8 relative in each of dx's and dW's summands, with signs that differ: their sum is off by 1.9e-3 in the norm, of which the result's own
// rounding is 1.7e-3), row-major and transposed, then both gradients in one launch.  Recomputing the logits is a quarter of the
// step's products; keeping them would be tokens x vocab.
//
// The products are c[m, n] = sum_k a[m, k] b[n, k] in bf16, v_mfma_f32_16x16x32_bf16, eight waves a workgroup.  64 values of k are 128
// bytes of a row: such slabs go to LDS by direct loads (rows past the end read as zeros), their 16-byte chunks swizzled by row, so that fragments
// are read without bank conflicts.  The rows of a slab are permuted on their way so that a lane's sums are four neighbouring rows by
// eight neighbouring columns: results leave as 16 bytes of a row, transposed ones as 8 bytes of a column, without a pass through LDS.
// x's gradient contracts over the weight's rows; it takes the weight as it lies, slabs of 64 rows of k, by transposing reads of LDS.
//
//   256 x 256 tiles (`ce_gemm_kernel`): 64 x 128 a wave; two slabs of a and three of b, one barrier per slab in the middle of its products.
//   64 or 128 x 64, 128 or 256 (`ce_gemm_ring_kernel`): few tokens, or few tiles; three to eight slabs of both in a ring.
//
// Bound by the matrix units where there are many tokens, and there by the board's power: 4096 tokens, 7168, 131072: forward 5.35 to 5.54 ms, 1.39 to 1.44
// PFLOP/s (hipBLASLt's product alone 1.46), backward 17.3 ms for three such products.  With few tokens by the weight's way from memory: 5 tokens
// 300 us, 6.2 TB/s.  In between by tiles' starts and ends: 512 tokens, 4096, 32000: 112 us, 1.20 PFLOP/s, and 406 us for the backward.
// One workgroup per compute unit with a list of tiles, whose first slabs arrive during the last ones of the tile before, was no
// faster (1531 tokens, 2048, 50001: 288 / 284 us forward, 535 / 540 the gradients) and slower where there is much work (gradients of a piece of
// 4096, 7168, 16384: 3.07 / 2.84 ms): the next tile's first wait includes the results' stores, and fixed lists do not even out.
#include <utility>

#include "gemm_tile.h"
#include "hpfp8_host.h"

namespace hpfp8 {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4_st __attribute__((ext_vector_type(4)));

constexpr int kTile = 256;
constexpr int kSlab = 64;                     // values of k in a slab: 128 bytes of a row
constexpr int kSlabBytes = kTile * 2 * kSlab;
constexpr float kLog2e = 1.44269504f;

constexpr int64_t kPieceElements = 0x3FFFF000;      // of a piece of the weight: its bytes are addressed with 31 bits

enum Epilogue { kStats = 0, kDlogits = 1, kGrads = 2 };
enum Store { kBf16 = 0, kF32 = 1, kF32Add = 2 };

// One product c[M, N] = a[M, K] b[N, K]^T; lda and ldb in bytes.
struct Product {
  const uint8_t* a;
  const uint8_t* b;
  int64_t lda, ldb;
  int M, N, K;
  void* c;
  int64_t ldc;           // elements
  int store;
  int tiles;
  int b_by_k;            // b is [K, N]
  int splits;            // parts of k, each with a c of its own, M ldc elements behind the one before
};

struct CeParams {
  Product part[2];       // (kGrads: two products that share the grid; otherwise the first alone)
  // kStats
  float2* stats;         // [M][parts] largest logit and sum of each tile of N
  int parts;
  float* sums;           // the same for the sum of the logits, or null
  float* target_logit;   // [M]
  // kStats and kDlogits
  const int64_t* target; // [M]
  int64_t rows_padded;   // stride of dl_t
  // kDlogits and kGrads: the gradient of the loss, one value, or one for each row with stride grad_stride
  const float* grad;
  int64_t grad_stride;
  const float* count;    // rows that count, when the loss is their mean; null otherwise
  // kDlogits
  const float* lse;      // [M]
  int64_t ignore_index;
  float smoothing;
  int64_t vocab;         // the whole of it
  int64_t first;         // the piece's first column
  uint16_t* dl;          // [rows_padded][ld_dl]
  int64_t ld_dl;
  uint16_t* dl_t;        // [N padded][rows_padded]
};

// Tile number -> (m tile, n tile): consecutive numbers cover rectangles of 32 tiles, an XCD's compute units at any moment, so that its L2
// serves each slab to several of them; the longer side of the rectangle goes along the shorter side of the grid.
__device__ __forceinline__ void tile_at(int t, int tiles_m, int tiles_n, int& tm, int& tn) {
  const int gm = tiles_m > tiles_n ? 4 : 8, gn_full = 32 / gm;
  const int per = gn_full * tiles_m;
  const int ng = t / per, rest = t - ng * per;
  const int gn = tiles_n - ng * gn_full < gn_full ? tiles_n - ng * gn_full : gn_full;
  const int mg = rest / (gm * gn), r = rest - mg * gm * gn;
  tm = mg * gm + r / gn;
  tn = ng * gn_full + r % gn;
}

// The XCD that a workgroup runs on gets a contiguous run of the tiles.
__device__ __forceinline__ int tile_of_workgroup(int pid, int tiles) {
  const int xcd = pid % kXcds, i = pid / kXcds, base = tiles / kXcds, more = tiles % kXcds;
  return xcd * base + (xcd < more ? xcd : more) + i;
}

// column (of the wave's 128) of sum r of subtile i in the lanes of group g, and the row of b that therefore goes to row p of LDS
__device__ __forceinline__ int column_of(int i, int g, int r) { return 32 * (i >> 1) + 8 * g + 4 * (i & 1) + r; }

// an operand's rows from `base` to its last one: a transfer from behind it reads zeros.  (A row ends with a whole 16-byte chunk: the workspaces
// whose length is none hold zeros there.)
__device__ __forceinline__ __amdgpu_buffer_rsrc_t resource(const uint8_t* base, int64_t rows, int64_t ld, int K) {
  const int64_t bytes = (rows - 1) * ld + (int64_t)((K + 7) & ~7) * 2;
  return __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, (int)(bytes < 0x7FFFF000 ? bytes : 0x7FFFF000), 0x00020000);
}
// 32 values of k out of a fragment's 64
__device__ __forceinline__ bf16x8 half_of(const v8i& f, int h) {
  return __builtin_bit_cast(bf16x8, v4i{f[4 * h], f[4 * h + 1], f[4 * h + 2], f[4 * h + 3]});
}

// The end of a tile of TM x TN: lane (l16, g) of a wave has the sums of rows m + j and columns n + column_of(i, g, r).
template <int EPI, int NS, int TM, int TN>
__device__ __forceinline__ void finish_tile(const CeParams& p, const Product& q, v4f (&acc)[NS][4], int m0, int n0, int m, int n, int g, uint8_t* lds) {
  const bool cut = n + 16 * NS > q.N;          // columns behind the end (their sums are zeros)
  if constexpr (EPI == kStats) {
    float2 out[4];
    float total[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t t = m + j < q.M ? p.target[m + j] : -1;
      const int own = t >= 0 && t < q.N ? (int)t : -1;
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < NS; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int c = n + column_of(i, g, r);
          if (cut && c >= q.N) acc[i][j][r] = -INFINITY;
          top = fmaxf(top, acc[i][j][r]);
          if (own == c) p.target_logit[m + j] = acc[i][j][r];
        }
      top = fmaxf(top, __shfl_xor(top, 16));
      top = fmaxf(top, __shfl_xor(top, 32));
      const float from = top == -INFINITY ? 0.f : top;      // (nothing but -inf: the sum is 0)
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < NS; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) sum += __builtin_amdgcn_exp2f((acc[i][j][r] - from) * kLog2e);
      sum += __shfl_xor(sum, 16);
      sum += __shfl_xor(sum, 32);
      out[j] = make_float2(top, sum);
      if (p.sums) {
        float all = 0.f;
#pragma unroll
        for (int i = 0; i < NS; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) all += cut && n + column_of(i, g, r) >= q.N ? 0.f : acc[i][j][r];
        all += __shfl_xor(all, 16);
        all += __shfl_xor(all, 32);
        total[j] = all;
      }
    }
    // the waves that share these rows, joined in LDS
    __syncthreads();
    float4* const each = reinterpret_cast<float4*>(lds);          // [waves along n][rows of the tile]
    if (g == 0) {
#pragma unroll
      for (int j = 0; j < 4; ++j) each[(n - n0) / (16 * NS) * TM + m - m0 + j] = make_float4(out[j].x, out[j].y, p.sums ? total[j] : 0.f, 0.f);
    }
    __syncthreads();
    const int row = m0 + (int)threadIdx.x;
    if ((int)threadIdx.x < TM && row < q.M) {
      float top = -INFINITY, sum = 0.f, all = 0.f;
#pragma unroll
      for (int k = 0; k < TN / (16 * NS); ++k) top = fmaxf(top, each[k * TM + threadIdx.x].x);
      const float from = top == -INFINITY ? 0.f : top;
#pragma unroll
      for (int k = 0; k < TN / (16 * NS); ++k) {
        const float4 v = each[k * TM + threadIdx.x];
        sum += v.y * __builtin_amdgcn_exp2f((v.x - from) * kLog2e);
        all += v.z;
      }
      const int64_t at = (int64_t)row * p.parts + n0 / TN;
      p.stats[at] = make_float2(top, sum);
      if (p.sums) p.sums[at] = all;
    }
  } else if constexpr (EPI == kDlogits) {
    const float flat = p.smoothing / (float)p.vocab, one = 1.0f - p.smoothing;
    uint32_t pk[4][NS][2];                      // [j][i][r / 2]: bf16 pairs along the columns
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool row = m + j < q.M;
      const int64_t t = row ? p.target[m + j] : p.ignore_index;
      float c = 0.f, lse = 0.f;
      if (t != p.ignore_index) {
        lse = p.lse[m + j];
        c = p.grad_stride ? p.grad[(int64_t)(m + j) * p.grad_stride] : 1.f;
        if (t < 0 || t >= p.vocab) c = NAN;
      }
      const int own = t >= p.first && t < p.first + q.N ? (int)(t - p.first) : -1;
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        float d[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int col = n + column_of(i, g, r);
          float v = __builtin_amdgcn_exp2f((acc[i][j][r] - lse) * kLog2e) - flat;
          if (own == col) v -= one;
          d[r] = t == p.ignore_index || (cut && col >= q.N) ? 0.f : c * v;
        }
        pk[j][i][0] = pack_bf16x2(d[0], d[1]);
        pk[j][i][1] = pack_bf16x2(d[2], d[3]);
      }
#pragma unroll
      for (int h = 0; h < NS / 2; ++h) {
        const u32x4_st v = {pk[j][2 * h][0], pk[j][2 * h][1], pk[j][2 * h + 1][0], pk[j][2 * h + 1][1]};
        *reinterpret_cast<u32x4_st*>(p.dl + (int64_t)(m + j) * p.ld_dl + n + 32 * h + 8 * g) = v;
      }
    }
#pragma unroll
    for (int i = 0; i < NS; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const uint32_t sel = r & 1 ? 0x07060302u : 0x05040100u;       // the upper or the lower halves of two words
        uint2 v;
        v.x = __builtin_amdgcn_perm(pk[1][i][r >> 1], pk[0][i][r >> 1], sel);
        v.y = __builtin_amdgcn_perm(pk[3][i][r >> 1], pk[2][i][r >> 1], sel);
        *reinterpret_cast<uint2*>(p.dl_t + (int64_t)(n + column_of(i, g, r)) * p.rows_padded + m) = v;
      }
  } else {
    if (p.grad) {
      // (one factor for all rows is applied here, so that what was rounded is a difference of probabilities: of c (p - 1) the most
      // frequent value by far, -c, would be rounded the same way in every row)
      // (the mean over no rows is NaN, but no row has a part in it: its gradient is 0)
      const float rows = p.count ? p.count[0] : 1.f, c = rows > 0.f ? p.grad[0] / rows : 0.f;
#pragma unroll
      for (int i = 0; i < NS; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] *= c;
    }
    if (q.store == kBf16) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (m + j >= q.M) break;
        uint16_t* const row = reinterpret_cast<uint16_t*>(q.c) + (int64_t)(m + j) * q.ldc;
#pragma unroll
        for (int h = 0; h < NS / 2; ++h) {
          const int col = n + 32 * h + 8 * g;
          const u32x4_st v = {pack_bf16x2(acc[2 * h][j][0], acc[2 * h][j][1]), pack_bf16x2(acc[2 * h][j][2], acc[2 * h][j][3]),
                              pack_bf16x2(acc[2 * h + 1][j][0], acc[2 * h + 1][j][1]), pack_bf16x2(acc[2 * h + 1][j][2], acc[2 * h + 1][j][3])};
          if (col < q.N) *reinterpret_cast<u32x4_st*>(row + col) = v;
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (m + j >= q.M) break;
        float* const row = reinterpret_cast<float*>(q.c) + (int64_t)(m + j) * q.ldc;
#pragma unroll
        for (int i = 0; i < NS; ++i) {
          const int col = n + (q.b_by_k ? 16 * i + 4 * g : column_of(i, g, 0));
          if (col >= q.N) continue;
          v4f v = acc[i][j];
          if (q.store == kF32Add) v += *reinterpret_cast<const v4f*>(row + col);
          *reinterpret_cast<v4f*>(row + col) = v;
        }
      }
    }
  }
}

// Slabs of a b that lies with its rows along k (BT) are 64 rows of 512 bytes, in 32-byte slots swizzled so that the eight rows that half a
// wave reads at a time lie in different banks.
typedef int i32x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ int slot_swizzle(int k) { return (k & 3) | (k >> 4 & 1) << 2; }

// The sums of a tile.  BT: b is [K, N], its rows along k; its fragments are then gathered by transposing reads, and subtile i is columns
// 16 i ... instead of column_of's.
template <bool BT>
__device__ __forceinline__ void multiply(const Product& q, int m0, int n0, uint8_t* lds, int lane, int wave, v4f (&acc)[8][4]) {
  uint8_t* const a_lds = lds;
  uint8_t* const b_lds = lds + 2 * kSlabBytes;
  const int slabs = (q.K + kSlab - 1) / kSlab;
  // ---- transfers: one is 8 rows x 128 bytes of LDS per wave, four per wave and slab
  const __amdgpu_buffer_rsrc_t rsrc_a = resource(q.a + (int64_t)m0 * q.lda, q.M - m0, q.lda, q.K);
  const __amdgpu_buffer_rsrc_t rsrc_b = BT ? resource(q.b + (int64_t)n0 * 2, q.K, q.ldb, q.N - n0) : resource(q.b + (int64_t)n0 * q.ldb, q.N - n0, q.ldb, q.K);
  uint32_t a_off[4], b_off[4], past[2], past_b[BT ? 4 : 1];
  const int whole = q.K / kSlab;               // slabs that are not cut off by the end of k
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = (wave * 4 + i) * 8 + (lane >> 3);
    const int chunk = (lane & 7) ^ row_swizzle(r);
    const int ra = (r & ~63) + (r & 15) * 4 + ((r >> 4) & 3);
    const int rb = (r & ~127) + column_of((r >> 4) & 7, (r >> 2) & 3, r & 3);
    a_off[i] = (uint32_t)ra * (uint32_t)q.lda + chunk * 16;
    b_off[i] = (uint32_t)rb * (uint32_t)q.ldb + chunk * 16;
    if constexpr (BT) {
      const int k = (wave * 4 + i) * 2 + (lane >> 5);       // 2 rows x 512 bytes
      b_off[i] = (uint32_t)k * (uint32_t)q.ldb + (((lane & 31) >> 1 ^ slot_swizzle(k)) * 2 + (lane & 1)) * 16;
      past_b[i] = k >= q.K % kSlab ? 0x80000000u : 0u;
    }
    // (a chunk behind the end of k is read from beyond the resource, as zeros; the swizzle has two patterns over i)
    if (i < 2) past[i] = chunk * 8 >= q.K % kSlab ? 0x80000000u : 0u;
  }
  const int b_step = BT ? kSlab * (int)q.ldb : 128;
  auto load = [&](const __amdgpu_buffer_rsrc_t& rs, uint32_t off, uint32_t behind, uint8_t* to, int slab, int step, int i) {
    // (behind the last slab the last one again: those are never used)
    const int s = slab < slabs ? slab : slabs - 1;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_ptr_t)(to + (wave * 4 + i) * 1024), 16, off + (s >= whole ? behind : 0u), s * step, 0, 0);
  };
  auto load_a = [&](int buf, int slab, int i) { load(rsrc_a, a_off[i], past[i & 1], a_lds + buf * kSlabBytes, slab, 128, i); };
  auto load_b = [&](int buf, int slab, int i) {
    load(rsrc_b, b_off[i], BT ? past_b[i] : past[i & 1], b_lds + buf * kSlabBytes, slab, b_step, i);
  };

  const int wn = wave & 1, wm = wave >> 1, l16 = lane & 15, g = lane >> 4;
  int frag_lo = l16 * 128 + ((2 * g) ^ row_swizzle(l16)) * 16, frag_hi = frag_lo ^ 16;
  asm volatile("" : "+v"(frag_lo), "+v"(frag_hi));
  const int a_frag = wm * 64 * 128, b_frag = wn * 128 * 128;
  // BT: a lane's 8 bytes of four rows of k; the group's 16 lanes exchange them, so that each has four values of k of one column.  (Through the
  // builtin every such read waits for all transfers under way.  The reads of two subtiles and their wait are one block.)
  const uint32_t tr_row = (16 * g + (l16 >> 2)) * 512 + (l16 & 3) * 8 + (uint32_t)(uintptr_t)(lds_ptr_t)lds, tr_slot = slot_swizzle(16 * g + (l16 >> 2)) * 32;
  auto read_two = [&](const uint8_t* slab, int i, v8i& f0, v8i& f1) {
    const uint32_t at = tr_row + (uint32_t)(slab - lds);
    const uint32_t at0 = at + (((wn * 8 + i) * 32) ^ tr_slot), at1 = at + (((wn * 8 + i + 1) * 32) ^ tr_slot);
    i32x2 r[8];
    asm volatile(
        "ds_read_b64_tr_b16 %0, %8\n\tds_read_b64_tr_b16 %1, %8 offset:2048\n\tds_read_b64_tr_b16 %2, %8 offset:4096\n\t"
        "ds_read_b64_tr_b16 %3, %8 offset:6144\n\tds_read_b64_tr_b16 %4, %9\n\tds_read_b64_tr_b16 %5, %9 offset:2048\n\t"
        "ds_read_b64_tr_b16 %6, %9 offset:4096\n\tds_read_b64_tr_b16 %7, %9 offset:6144\n\ts_waitcnt lgkmcnt(0)"
        : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3]), "=&v"(r[4]), "=&v"(r[5]), "=&v"(r[6]), "=&v"(r[7])
        : "v"(at0), "v"(at1)
        : "memory");
    f0 = v8i{r[0][0], r[0][1], r[1][0], r[1][1], r[2][0], r[2][1], r[3][0], r[3][1]};
    f1 = v8i{r[4][0], r[4][1], r[5][0], r[5][1], r[6][0], r[6][1], r[7][0], r[7][1]};
  };
  auto read_b = [&](const uint8_t* slab, int i) { return frag_read(slab + b_frag + i * 16 * 128, frag_lo, frag_hi); };

  const v4f zero = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = zero;

  // ---- slab 0 of both, slab 1 of b, the first half of slab 1 of a
#pragma unroll
  for (int i = 0; i < 4; ++i) load_a(0, 0, i);
#pragma unroll
  for (int i = 0; i < 4; ++i) load_b(0, 0, i);
#pragma unroll
  for (int i = 0; i < 4; ++i) load_b(1, 1, i);
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_waitcnt(0x0F70 | 4);      // all but the last four have landed
  __syncthreads();
  load_a(1, 1, 0);
  load_a(1, 1, 1);

  v8i xf[4], wf[4];
  if constexpr (BT) read_two(b_lds, 0, wf[0], wf[1]);
  else wf[0] = read_b(b_lds, 0);
#pragma unroll
  for (int j = 0; j < 4; ++j) xf[j] = frag_read(a_lds + a_frag + j * 16 * 128, frag_lo, frag_hi);
  if (!BT) wf[1] = read_b(b_lds, 1);

  // One slab.  Its barrier sits before its last two subtiles: what follows it, the fragments of the next slab, is covered by the matrix
  // instructions that are left.  Transfers, one per subtile: the rest of the next slab of a, the slab after next of b, and behind
  // the barrier the first half of the slab after next of a into the buffer that every wave has just left.
  int abuf = 0, bbuf = 0;
  for (int s = 0; s < slabs; ++s) {
    const int bnext = bbuf == 2 ? 0 : bbuf + 1, bnew = bnext == 2 ? 0 : bnext + 1;
    const uint8_t* const bcur = b_lds + bbuf * kSlabBytes;
    const uint8_t* const bnxt = b_lds + bnext * kSlabBytes;
    const uint8_t* const anxt = a_lds + (abuf ^ 1) * kSlabBytes;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (i == 6) {
        __builtin_amdgcn_s_waitcnt(0x0070 | 4);         // vmcnt(4) lgkmcnt(0): b's slab after next may be under way
        __builtin_amdgcn_s_barrier();
      }
      if constexpr (!BT) wf[(i + 2) % 4] = i < 6 ? read_b(bcur, i + 2) : read_b(bnxt, i - 6);
      else if (i % 2 == 0) read_two(i < 6 ? bcur : bnxt, i < 6 ? i + 2 : 0, wf[(i + 2) % 4], wf[(i + 3) % 4]);
      if (i < 2) load_a(abuf ^ 1, s + 1, i + 2);
      else if (i < 6) load_b(bnew, s + 2, i - 2);
      else load_a(abuf, s + 2, i - 6);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(half_of(wf[i % 4], 0), half_of(xf[j], 0), acc[i][j], 0, 0, 0);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(half_of(wf[i % 4], 1), half_of(xf[j], 1), acc[i][j], 0, 0, 0);
        if (i == 7) xf[j] = frag_read(anxt + a_frag + j * 16 * 128, frag_lo, frag_hi);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    abuf ^= 1;
    bbuf = bnext;
  }
  __builtin_amdgcn_s_waitcnt(0x0F70);          // vmcnt(0): the last transfers write to this workgroup's LDS
}

template <int EPI>
__global__ __launch_bounds__(512) void ce_gemm_kernel(CeParams p) {
  __shared__ __attribute__((aligned(1024))) uint8_t lds[5 * kSlabBytes];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int pid = blockIdx.x;
  const int before = EPI == kGrads ? p.part[0].tiles * p.part[0].splits : 0;
  const bool second = EPI == kGrads && pid >= before;
  Product q = second ? p.part[1] : p.part[0];
  int t = tile_of_workgroup(second ? pid - before : pid, q.tiles * q.splits), tm, tn;
  if (EPI == kGrads && q.splits > 1) {
    const int split = t / q.tiles, all = (q.K + kSlab - 1) / kSlab;
    t -= split * q.tiles;
    const int from = (int)((int64_t)all * split / q.splits), to = (int)((int64_t)all * (split + 1) / q.splits);
    q.a += (int64_t)from * kSlab * 2;
    q.b += (int64_t)from * kSlab * (q.b_by_k ? q.ldb : 2);
    q.K = (to < all ? to * kSlab : q.K) - from * kSlab;
    q.c = reinterpret_cast<float*>(q.c) + (int64_t)split * q.M * q.ldc;
  }
  tile_at(t, (q.M + kTile - 1) / kTile, (q.N + kTile - 1) / kTile, tm, tn);
  const int m0 = tm * kTile, n0 = tn * kTile;
  v4f acc[8][4];
  if (EPI == kGrads && q.b_by_k) multiply<true>(q, m0, n0, lds, lane, wave, acc);
  else multiply<false>(q, m0, n0, lds, lane, wave, acc);
  finish_tile<EPI, 8, kTile, kTile>(p, q, acc, m0, n0, m0 + (wave >> 1) * 64 + (lane & 15) * 4, n0 + (wave & 1) * 128, lane >> 4, lds);
}

// All but this wave's last LEFT transfers have landed, and what it has read of LDS is in its registers (behind the barrier a transfer of any wave may
// take the place of what was read); then all waves'.
template <int LEFT>
__device__ __forceinline__ void wait_and_meet() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(LEFT) : "memory");
}

// Smaller tiles: 64 WM rows and COLS columns in WM x WN waves, each with 64 rows and 32 or 64 columns, so that few tokens or a small vocabulary
// give more compute units a tile.  LDS is a ring of slabs of both operands, on their way while another one is multiplied; one barrier per slab.
constexpr int ring_stages(int rows, int cols) { return cols == 64 ? 8 : cols == 128 ? (rows == 64 ? 6 : 5) : (rows == 64 ? 4 : 3); }
template <int EPI, int WM, int WN, int COLS>
__device__ __forceinline__ void ring_tile(const CeParams& p, uint8_t* lds) {
  constexpr int kRows = 64 * WM, kCols = COLS, NS = kCols / (16 * WN), kStages = ring_stages(kRows, kCols), kStage = (kRows + kCols) * 128;
  constexpr int kLoadsA = 8 / WN, kLoadsB = kCols / (8 * WM * WN);      // a wave's transfers of a slab
  constexpr int kLeft = (kStages - 2) * (kLoadsA + kLoadsB);            // transfers of the slabs behind the next one
  // a slab's fragments are read while the one before is multiplied, at the price of one slab fewer on its way (64 x 64 tiles, 16 tokens, 6592,
  // 2859 41 / 35 us; 64 x 256 ones, 506, 6328, 5743 120 / 115)
  constexpr bool kReadAhead = kStages > 3;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Product q = p.part[0];
  int tm, tn;
  tile_at(tile_of_workgroup(blockIdx.x, q.tiles), (q.M + kRows - 1) / kRows, (q.N + kCols - 1) / kCols, tm, tn);
  const int m0 = tm * kRows, n0 = tn * kCols, slabs = (q.K + kSlab - 1) / kSlab, whole = q.K / kSlab;
  const __amdgpu_buffer_rsrc_t rsrc_a = resource(q.a + (int64_t)m0 * q.lda, q.M - m0, q.lda, q.K);
  const __amdgpu_buffer_rsrc_t rsrc_b = resource(q.b + (int64_t)n0 * q.ldb, q.N - n0, q.ldb, q.K);
  uint32_t a_off[kLoadsA], b_off[kLoadsB], past[2];
  auto chunk_of = [&](int r) { return (lane & 7) ^ row_swizzle(r); };
#pragma unroll
  for (int i = 0; i < kLoadsA; ++i) {
    const int r = (wave * kLoadsA + i) * 8 + (lane >> 3);
    a_off[i] = (uint32_t)((r & ~63) + (r & 15) * 4 + ((r >> 4) & 3)) * (uint32_t)q.lda + chunk_of(r) * 16;
  }
#pragma unroll
  for (int i = 0; i < kLoadsB; ++i) {
    const int r = (wave * kLoadsB + i) * 8 + (lane >> 3);
    b_off[i] = (uint32_t)((r & ~(16 * NS - 1)) + column_of((r >> 4) & (NS - 1), (r >> 2) & 3, r & 3)) * (uint32_t)q.ldb + chunk_of(r) * 16;
    // (a chunk behind the end of k is read from beyond the resource, as zeros; the swizzle has two patterns, by whether r / 8 is odd)
    if (i < 2) past[i] = chunk_of(r) * 8 >= q.K % kSlab ? 0x80000000u : 0u;
  }
  auto load = [&](int slab) {
    uint8_t* const to = lds + slab % kStages * kStage;
    const int s = slab < slabs ? slab : slabs - 1;        // (behind the last slab the last one again: those are never used)
    const bool cut = s >= whole;
#pragma unroll
    for (int i = 0; i < kLoadsA; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc_a, (lds_ptr_t)(to + (wave * kLoadsA + i) * 1024), 16, a_off[i] + (cut ? past[(wave * kLoadsA + i) & 1] : 0u),
                                               s * 128, 0, 0);
#pragma unroll
    for (int i = 0; i < kLoadsB; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc_b, (lds_ptr_t)(to + kRows * 128 + (wave * kLoadsB + i) * 1024), 16, b_off[i] + (cut ? past[i & 1] : 0u),
                                               s * 128, 0, 0);
  };
  const int wm = wave / WN, wn = wave % WN, l16 = lane & 15, g = lane >> 4;
  const int frag_lo = l16 * 128 + ((2 * g) ^ row_swizzle(l16)) * 16, frag_hi = frag_lo ^ 16;
  const v4f zero = {0.f, 0.f, 0.f, 0.f};
  v4f acc[NS][4];
#pragma unroll
  for (int i = 0; i < NS; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = zero;
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) load(s);
  v8i wf[kReadAhead ? 2 : 1][NS], xf[kReadAhead ? 2 : 1][4];
  auto read = [&](v8i (&w)[NS], v8i (&x)[4], int s) {
    const uint8_t* const a = lds + s % kStages * kStage + wm * 64 * 128;
    const uint8_t* const b = lds + s % kStages * kStage + kRows * 128 + wn * 16 * NS * 128;
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = frag_read(a + j * 16 * 128, frag_lo, frag_hi);
#pragma unroll
    for (int i = 0; i < NS; ++i) w[i] = frag_read(b + i * 16 * 128, frag_lo, frag_hi);
  };
  auto multiply_slab = [&](const v8i (&w)[NS], const v8i (&x)[4]) {
#pragma unroll
    for (int i = 0; i < NS; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(half_of(w[i], h), half_of(x[j], h), acc[i][j], 0, 0, 0);
  };
  if constexpr (kReadAhead) {
    wait_and_meet<kLeft>();
    read(wf[0], xf[0], 0);
    auto step = [&](int s, int u) {
      // slab s + 1 is there, and slab s - 1 has been multiplied by all: its place takes the next transfers
      wait_and_meet<kLeft - kLoadsA - kLoadsB>();
      load(s + kStages - 1);
      read(wf[u ^ 1], xf[u ^ 1], s + 1);
      multiply_slab(wf[u], xf[u]);
    };
    for (int s = 0; s < slabs; s += 2) {
      step(s, 0);
      if (s + 1 < slabs) step(s + 1, 1);
    }
  } else {
    for (int s = 0; s < slabs; ++s) {
      // slab s is there (those after it may be under way), and the one before has been read by all
      wait_and_meet<kLeft>();
      load(s + kStages - 1);
      read(wf[0], xf[0], s);
      multiply_slab(wf[0], xf[0]);
    }
  }
  __builtin_amdgcn_s_waitcnt(0x0F70);          // vmcnt(0): the last transfers write to this workgroup's LDS
  finish_tile<EPI, NS, kRows, kCols>(p, q, acc, m0, n0, m0 + wm * 64 + l16 * 4, n0 + wn * 16 * NS, g, lds);
}
template <int EPI, int WM, int WN, int COLS>
__global__ __launch_bounds__(64 * WM * WN) void ce_gemm_ring_kernel(CeParams p) {
  __shared__ __attribute__((aligned(1024))) uint8_t lds[ring_stages(64 * WM, COLS) * (64 * WM + COLS) * 128];
  ring_tile<EPI, WM, WN, COLS>(p, lds);
}

// ---- joins the forward's partial results, a wave for each row
__global__ __launch_bounds__(256) void ce_join_kernel(const float2* __restrict__ stats, const float* __restrict__ sums,
                                                      const float* __restrict__ target_logit, const int64_t* __restrict__ target, int parts,
                                                      int64_t rows, int64_t ignore_index, int64_t vocab, float smoothing, float* __restrict__ lse,
                                                      float* __restrict__ loss) {
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= rows) return;
  const float2* const s = stats + row * parts;
  float top = -INFINITY, sum = 0.f, total = 0.f;
  auto add = [&](float2 v) {
    const float t = fmaxf(top, v.x), from = t == -INFINITY ? 0.f : t;
    sum = sum * __builtin_amdgcn_exp2f((top - from) * kLog2e) + v.y * __builtin_amdgcn_exp2f((v.x - from) * kLog2e);
    top = t;
  };
  int k = lane;
  for (; k + 448 < parts; k += 512) {
    float2 v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) v[u] = s[k + 64 * u];
#pragma unroll
    for (int u = 0; u < 8; ++u) add(v[u]);
  }
  for (; k < parts; k += 64) add(s[k]);
  if (sums)
    for (k = lane; k < parts; k += 64) total += sums[row * parts + k];
  for (int d = 1; d < 64; d *= 2) {
    add(make_float2(__shfl_xor(top, d), __shfl_xor(sum, d)));
    total += __shfl_xor(total, d);
  }
  if (lane != 0) return;
  const float l = (top == -INFINITY ? 0.f : top) + logf(sum);
  if (lse) lse[row] = l;
  const int64_t t = target[row];
  float out = 0.f;
  if (t != ignore_index) {
    out = t < 0 || t >= vocab ? NAN : l - (1.0f - smoothing) * target_logit[row];
    if (smoothing != 0.f) out -= smoothing * (total / (float)vocab);
  }
  loss[row] = out;
}

// ---- the rows' losses, their sum or mean, and how many count: one workgroup, in a fixed order
__global__ __launch_bounds__(1024) void ce_reduce_kernel(const float* __restrict__ loss, const int64_t* __restrict__ target, int64_t rows,
                                                         int64_t ignore_index, int mean, float* __restrict__ out, float* __restrict__ count) {
  __shared__ double sums[16];
  __shared__ int64_t counts[16];
  double s = 0.0;
  int64_t n = 0;
  for (int64_t r = threadIdx.x; r < rows; r += 1024) {
    s += (double)loss[r];
    n += target[r] != ignore_index;
  }
  for (int d = 1; d < 64; d *= 2) {
    s += __shfl_xor(s, d);
    n += __shfl_xor(n, d);
  }
  if ((threadIdx.x & 63) == 0) {
    sums[threadIdx.x >> 6] = s;
    counts[threadIdx.x >> 6] = n;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    s = 0.0;
    n = 0;
    for (int k = 0; k < 16; ++k) {
      s += sums[k];
      n += counts[k];
    }
    *out = (float)(mean ? s / (double)n : s);
    *count = (float)n;
  }
}

// ---- out[c, r] = in[r, c], bf16, 64 x 64 per workgroup; columns of out from rows to the next multiple of 64 are zeros, and so are those of
// rows whose target is ignored (what such a row holds, NaN in padding too, then meets a gradient of 0 as 0)
__global__ __launch_bounds__(256) void ce_transpose_kernel(const uint16_t* __restrict__ in, int64_t ld, int64_t rows, int64_t cols,
                                                           const int64_t* __restrict__ target, int64_t ignore_index, uint16_t* __restrict__ out,
                                                           int64_t ld_out) {
  __shared__ uint16_t tile[64][66];
  const int64_t r0 = (int64_t)blockIdx.x * 64, c0 = (int64_t)blockIdx.y * 64;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = threadIdx.x / 8 + 32 * h, c = threadIdx.x % 8 * 8;
    u32x4_st v = {0, 0, 0, 0};
    if (r0 + r < rows && c0 + c < cols && !(target && target[r0 + r] == ignore_index)) v = *reinterpret_cast<const u32x4_st*>(in + (r0 + r) * ld + c0 + c);
#pragma unroll
    for (int k = 0; k < 4; ++k) *reinterpret_cast<uint32_t*>(&tile[r][c + 2 * k]) = v[k];
  }
  __syncthreads();
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int c = threadIdx.x / 8 + 32 * h, r = threadIdx.x % 8 * 8;
    if (c0 + c >= cols) continue;
    u32x4_st v;
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = (uint32_t)tile[r + 2 * k][c] | (uint32_t)tile[r + 2 * k + 1][c] << 16;
    *reinterpret_cast<u32x4_st*>(out + (c0 + c) * ld_out + r0 + r) = v;
  }
}

// ---- the sum of the parts, in order, rounded to bf16
__global__ __launch_bounds__(256) void ce_round_kernel(const float* __restrict__ in, int64_t n8, int parts, uint16_t* __restrict__ out) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n8) return;
  const v4f* at = reinterpret_cast<const v4f*>(in) + 2 * i;
  v4f a = at[0], b = at[1];
  for (int k = 1; k < parts; ++k) {
    at += 2 * n8;
    a += at[0];
    b += at[1];
  }
  reinterpret_cast<u32x4_st*>(out)[i] = u32x4_st{pack_bf16x2(a[0], a[1]), pack_bf16x2(a[2], a[3]), pack_bf16x2(b[0], b[1]), pack_bf16x2(b[2], b[3])};
}

// ---- the weight's gradient of no tokens
__global__ __launch_bounds__(256) void ce_zero_kernel(u32x4_st* __restrict__ out, int64_t n16) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n16; i += (int64_t)gridDim.x * 256) out[i] = u32x4_st{0, 0, 0, 0};
}

// Elements between the rows of the workspaces: whole tiles, and an odd number of 128-byte lines, so that the rows of a tile do not all lie
// in the same few memory channels (the gradients' launch of 4096 tokens, 7168, 16384 columns: 1480 us with strides of 2^13 and 2^15 bytes).
int64_t up(int64_t n, int64_t to);
int64_t stride_of(int64_t n) { return up(n, kTile) + kSlab; }
int64_t up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }
int64_t tiles_of(int64_t m, int64_t n, int rows = kTile, int cols = kTile) { return (m + rows - 1) / rows * ((n + cols - 1) / cols); }

int check(int64_t tokens, int64_t hidden, int64_t vocab, int64_t ld_x, int64_t ld_w) {
  HPFP8_REQUIRE(tokens >= 0 && hidden > 0 && vocab > 0, HPFP8_ERR_SHAPE, "tokens=%lld hidden=%lld vocab=%lld", (long long)tokens, (long long)hidden, (long long)vocab);
  HPFP8_REQUIRE(hidden % 8 == 0 && ld_x % 8 == 0 && ld_w % 8 == 0, HPFP8_ERR_SHAPE, "hidden and the row strides must be multiples of 8");
  HPFP8_REQUIRE(ld_x >= hidden && ld_w >= hidden, HPFP8_ERR_SHAPE, "a row stride is below hidden");
  HPFP8_REQUIRE(ld_x < (1 << 21) && ld_w < (1 << 21), HPFP8_ERR_SHAPE, "rows of 4 MiB and more");
  // (256 rows of a workspace with a column for each token are addressed with 31 bits)
  HPFP8_REQUIRE(tokens <= (1 << 21) && vocab <= (1 << 24), HPFP8_ERR_SHAPE, "tokens=%lld vocab=%lld: at most 2^21 and 2^24", (long long)tokens, (long long)vocab);
  return HPFP8_OK;
}

Product product(const void* a, int64_t lda, const void* b, int64_t ldb, int64_t M, int64_t N, int64_t K, void* c, int64_t ldc, int store) {
  Product q = {};
  q.a = (const uint8_t*)a;
  q.b = (const uint8_t*)b;
  q.lda = lda * 2;
  q.ldb = ldb * 2;
  q.M = (int)M;
  q.N = (int)N;
  q.K = (int)K;
  q.c = c;
  q.ldc = ldc;
  q.store = store;
  q.tiles = (int)tiles_of(M, N);
  q.splits = 1;
  return q;
}

// The tile whose rounds on the compute units are the shortest, from what a slab of it takes and its start and end.  us of a forward with
//                          256 x 256 / 128 x 256 / 64 x 256 / 128 x 128 / 64 x 128 / 64 x 64
//   16 tokens, 6592, 2859    133 /  89 /  74 /  50 /  45 /  35        506, 6328, 5743     173 / 136 / 115 /  98 / 130 / 151
//   24, 1472, 33651           44 /  31 /  29 /  39 /  38 /  39        1014, 6784, 5994    138 / 100 / 132 / 118 / 134 / 200
//   100, 2048, 16000          53 /  39 /  34 /  29 /  26 /  35        3715, 1616, 4098     53 /  67 /  97 /  85 / 126 / 184
//   128, 4096, 32000         101 /  80 /  73 /  67 /  81 / 107        96, 4096, 131072    223 / 187 / 226 / 197 / 260 / 354
struct Form {
  int rows, cols;        // of a tile
  int slab, ends;        // 10 ns
};
constexpr Form kForms[] = {{256, 256, 125, 500}, {128, 256, 90, 400}, {64, 256, 70, 400}, {128, 128, 55, 350}, {64, 128, 38, 350}, {64, 64, 30, 300}};
Form form_of(int64_t tokens, int64_t hidden, int64_t vocab) {
  const int64_t slabs = (hidden + kSlab - 1) / kSlab;
  Form best = kForms[0];
  int64_t least = INT64_MAX;
  for (const Form& f : kForms) {
    const int64_t cost = (tiles_of(tokens, vocab, f.rows, f.cols) + 255) / 256 * (f.slab * slabs + f.ends);
    if (cost < least) {
      least = cost;
      best = f;
    }
  }
  return best;
}
template <int EPI>
void launch_logits(CeParams& p, const Form& form, hipStream_t s) {
  Product& q = p.part[0];
  q.tiles = (int)tiles_of(q.M, q.N, form.rows, form.cols);
  if (form.cols == 64) ce_gemm_ring_kernel<EPI, 1, 2, 64><<<q.tiles, 128, 0, s>>>(p);
  else if (form.cols == 128 && form.rows == 64) ce_gemm_ring_kernel<EPI, 1, 4, 128><<<q.tiles, 256, 0, s>>>(p);
  else if (form.cols == 128) ce_gemm_ring_kernel<EPI, 2, 4, 128><<<q.tiles, 512, 0, s>>>(p);
  else if (form.rows == 64) ce_gemm_ring_kernel<EPI, 1, 8, 256><<<q.tiles, 512, 0, s>>>(p);
  else if (form.rows == 128) ce_gemm_ring_kernel<EPI, 2, 4, 256><<<q.tiles, 512, 0, s>>>(p);
  else ce_gemm_kernel<EPI><<<q.tiles, 512, 0, s>>>(p);
}

// The gradients' launch: dx's product contracts over the whole piece and has few tiles, so with few tokens a few of its tiles would still be at
// work long after dw's are done.  Its contraction is split, and the longer of the two kinds of work goes first.  This is the time that 256
// compute units need for both, in slabs; a tile's start and end cost about six.  us of the launch unsplit / split: 512 tokens, 4096, 32000
// 736 / 256, 1531, 2048, 50001 1112 / 541.
constexpr int64_t kEnds = 6;
int64_t dx_part(int64_t width, int64_t splits) { return ((width + kSlab - 1) / kSlab + splits - 1) / splits + kEnds; }
int64_t dw_tile(int64_t tokens) { return (tokens + kSlab - 1) / kSlab + kEnds; }
int64_t gradients_time(int64_t tokens, int64_t hidden, int64_t width, int64_t splits, int with_dw) {
  int64_t n1 = tiles_of(tokens, hidden) * splits, each1 = dx_part(width, splits), n2 = with_dw ? tiles_of(width, hidden) : 0, each2 = dw_tile(tokens);
  if (each2 > each1) {
    std::swap(n1, n2);
    std::swap(each1, each2);
  }
  const int64_t rounds = n1 / 256, rest = n1 % 256;
  // compute units that have finished the longer kind, `rest` of them one round later, take the shorter one as it comes
  auto holds = [&](int64_t t) {
    const int64_t early = t - rounds * each1, late = early - each1;
    return (256 - rest) * (early > 0 ? early / each2 : 0) + rest * (late > 0 ? late / each2 : 0) >= n2;
  };
  int64_t from = (rounds + (rest > 0)) * each1, to = from + (n2 + 255) / 256 * each2;
  while (from < to) {
    const int64_t t = (from + to) / 2;
    if (holds(t)) to = t;
    else from = t + 1;
  }
  return from;
}

}  // namespace
}  // namespace hpfp8

using namespace hpfp8;

extern "C" {

int64_t hpfp8_cross_entropy_parts(int64_t tokens, int64_t hidden, int64_t vocab) {
  if (tokens <= 0 || hidden <= 0 || vocab <= 0) return 0;
  const int cols = form_of(tokens, hidden, vocab).cols;
  return (vocab + cols - 1) / cols;
}
int64_t hpfp8_cross_entropy_splits(int64_t tokens, int64_t hidden, int64_t width, int with_dw) {
  if (tokens <= 0 || hidden <= 0 || width <= 0) return 1;
  const int64_t slabs = (width + kSlab - 1) / kSlab;
  int64_t best = 1, least = INT64_MAX;
  for (int64_t splits = 1; splits <= 32 && splits <= slabs; ++splits) {
    // (the parts are written, and read by the sum: so many slabs' time at 4 TB/s)
    const int64_t cost = gradients_time(tokens, hidden, width, splits, with_dw) + splits * tokens * hidden * 8 / 5000000;
    if (cost < least) {
      least = cost;
      best = splits;
    }
  }
  return best;
}
int64_t hpfp8_cross_entropy_stride(int64_t n) { return n > 0 ? stride_of(n) : 0; }

int hpfp8_linear_cross_entropy_forward(const void* x, int64_t ld_x, const void* w, int64_t ld_w, const int64_t* target, int64_t tokens,
                                       int64_t hidden, int64_t vocab, int64_t ignore_index, float smoothing, int reduction, float* stats,
                                       float* sums, float* target_logit, float* lse, float* loss, float* out, float* count,
                                       hpfp8_stream_t stream) {
  const int bad = check(tokens, hidden, vocab, ld_x, ld_w);
  if (bad != HPFP8_OK) return bad;
  HPFP8_REQUIRE(reduction >= 0 && reduction <= 2, HPFP8_ERR_ARG, "unknown reduction %d", reduction);
  HPFP8_REQUIRE(smoothing >= 0.f && smoothing <= 1.f, HPFP8_ERR_ARG, "label smoothing must be in [0, 1]");
  HPFP8_REQUIRE(reduction == 0 || (out && count), HPFP8_ERR_ARG, "null buffer");
  const hipStream_t s = (hipStream_t)stream;
  if (tokens > 0) {
    HPFP8_REQUIRE(x && w && target && stats && target_logit && loss && (smoothing == 0.f || sums), HPFP8_ERR_ARG, "null buffer");
    HPFP8_REQUIRE(aligned16(x) && aligned16(w) && aligned16(stats), HPFP8_ERR_ALIGN, "a buffer is not 16-byte aligned");
    CeParams p = {};
    p.part[0] = product(x, ld_x, w, ld_w, tokens, vocab, hidden, nullptr, 0, 0);
    p.stats = (float2*)stats;
    p.sums = smoothing != 0.f ? sums : nullptr;
    p.target_logit = target_logit;
    p.target = target;
    const Form form = form_of(tokens, hidden, vocab);
    p.parts = (int)((vocab + form.cols - 1) / form.cols);
    launch_logits<kStats>(p, form, s);
    int rc = check_launch("linear_cross_entropy_forward");
    if (rc != HPFP8_OK) return rc;
    ce_join_kernel<<<(unsigned)((tokens + 3) / 4), 256, 0, s>>>(p.stats, p.sums, target_logit, target, p.parts, tokens, ignore_index, vocab, smoothing,
                                                              lse, loss);
    rc = check_launch("linear_cross_entropy_forward (join)");
    if (rc != HPFP8_OK) return rc;
  }
  return reduction != 0 ? hpfp8_linear_cross_entropy_reduce(loss, target, tokens, ignore_index, reduction, out, count, stream) : HPFP8_OK;
}

int hpfp8_linear_cross_entropy_reduce(const float* loss, const int64_t* target, int64_t tokens, int64_t ignore_index, int reduction, float* out,
                                      float* count, hpfp8_stream_t stream) {
  HPFP8_REQUIRE(tokens >= 0, HPFP8_ERR_SHAPE, "tokens=%lld", (long long)tokens);
  HPFP8_REQUIRE(reduction == 1 || reduction == 2, HPFP8_ERR_ARG, "unknown reduction %d", reduction);
  HPFP8_REQUIRE(out && count && (tokens == 0 || (loss && target)), HPFP8_ERR_ARG, "null buffer");
  ce_reduce_kernel<<<1, 1024, 0, (hipStream_t)stream>>>(loss, target, tokens, ignore_index, reduction == 1, out, count);
  return check_launch("linear_cross_entropy_reduce");
}

int hpfp8_linear_cross_entropy_piece(const void* x, int64_t ld_x, const void* x_t, const void* w, int64_t ld_w, const int64_t* target,
                                     int64_t tokens, int64_t hidden, int64_t vocab, int64_t first, int64_t width, int64_t ignore_index,
                                     float smoothing, const float* lse, const float* grad, int64_t grad_stride, const float* count, void* dl,
                                     void* dl_t, float* dx, int splits, int dx_add, void* dw, int dw_type, int dw_add,
                                     hpfp8_stream_t stream) {
  const int bad = check(tokens, hidden, vocab, ld_x, ld_w);
  if (bad != HPFP8_OK) return bad;
  HPFP8_REQUIRE(first >= 0 && width > 0 && first + width <= vocab, HPFP8_ERR_SHAPE, "piece %lld + %lld of %lld", (long long)first, (long long)width, (long long)vocab);
  HPFP8_REQUIRE(dw_type == HPFP8_OUT_BF16 || dw_type == HPFP8_OUT_F32, HPFP8_ERR_ARG, "unknown output type %d", dw_type);
  HPFP8_REQUIRE(!dx || (splits >= 1 && splits <= 32), HPFP8_ERR_ARG, "dx in %d parts", splits);
  const int64_t slabs = (width + kSlab - 1) / kSlab;
  HPFP8_REQUIRE(!dx || dx_add || splits <= slabs, HPFP8_ERR_ARG, "dx in %d parts of %lld slabs", splits, (long long)slabs);
  HPFP8_REQUIRE(width <= (1 << 21), HPFP8_ERR_SHAPE, "a piece of %lld columns: at most 2^21", (long long)width);
  HPFP8_REQUIRE(width * ld_w < kPieceElements, HPFP8_ERR_SHAPE, "a piece of %lld rows of the weight spans 2 GiB or more", (long long)width);
  HPFP8_REQUIRE(!dw_add || dw_type == HPFP8_OUT_F32, HPFP8_ERR_ARG, "only fp32 is added onto");
  if (tokens == 0) {
    if (!dw || dw_add) return HPFP8_OK;
    HPFP8_REQUIRE(aligned16(dw), HPFP8_ERR_ALIGN, "a buffer is not 16-byte aligned");
    const int64_t size = dw_type == HPFP8_OUT_F32 ? 4 : 2, n16 = width * hidden * size / 16, blocks = (n16 + 255) / 256;
    ce_zero_kernel<<<(unsigned)(blocks < 4096 ? blocks : 4096), 256, 0, (hipStream_t)stream>>>((u32x4_st*)((uint8_t*)dw + first * hidden * size), n16);
    return check_launch("linear_cross_entropy_piece (no tokens)");
  }
  HPFP8_REQUIRE(x && w && target && lse && grad && dl && dl_t && (!dw == !x_t), HPFP8_ERR_ARG, "null buffer");
  HPFP8_REQUIRE(aligned16(x) && aligned16(w) && aligned16(dl) && aligned16(dl_t) && aligned16(x_t) && aligned16(dx) && aligned16(dw),
                HPFP8_ERR_ALIGN, "a buffer is not 16-byte aligned");
  const hipStream_t s = (hipStream_t)stream;
  const int64_t rows_padded = stride_of(tokens), cols_padded = stride_of(width);
  const uint16_t* const piece = (const uint16_t*)w + first * ld_w;
  CeParams p = {};
  p.part[0] = product(x, ld_x, piece, ld_w, tokens, width, hidden, nullptr, 0, 0);
  p.target = target;
  p.rows_padded = rows_padded;
  p.lse = lse;
  p.grad = grad;
  p.grad_stride = grad_stride;
  p.count = count;
  p.ignore_index = ignore_index;
  p.smoothing = smoothing;
  p.vocab = vocab;
  p.first = first;
  p.dl = (uint16_t*)dl;
  p.ld_dl = cols_padded;
  p.dl_t = (uint16_t*)dl_t;
  launch_logits<kDlogits>(p, form_of(tokens, hidden, width), s);
  int rc = check_launch("linear_cross_entropy_piece");
  if (rc != HPFP8_OK) return rc;
  CeParams g = {};
  int n = 0;
  if (dx) {
    g.part[n] = product(dl, cols_padded, piece, ld_w, tokens, hidden, width, dx, hidden, dx_add ? kF32Add : kF32);
    g.part[n].b_by_k = 1;
    g.part[n++].splits = (int)(splits < slabs ? splits : slabs);      // (a narrower piece adds onto fewer parts)
  }
  if (dw) {
    void* const to = (uint8_t*)dw + first * hidden * (dw_type == HPFP8_OUT_F32 ? 4 : 2);
    g.part[n++] = product(dl_t, rows_padded, x_t, rows_padded, width, hidden, up(tokens, kSlab), to, hidden,
                          dw_type == HPFP8_OUT_BF16 ? kBf16 : (dw_add ? kF32Add : kF32));
  }
  if (n == 0) return HPFP8_OK;
  if (n == 2 && dw_tile(tokens) > dx_part(width, splits)) std::swap(g.part[0], g.part[1]);
  g.grad = grad_stride ? nullptr : grad;
  g.count = count;
  ce_gemm_kernel<kGrads><<<g.part[0].tiles * g.part[0].splits + g.part[1].tiles * g.part[1].splits, 512, 0, s>>>(g);
  return check_launch("linear_cross_entropy_piece (gradients)");
}

int hpfp8_linear_cross_entropy_rows_t(const void* x, int64_t rows, int64_t cols, int64_t ld, const int64_t* target, int64_t ignore_index, void* x_t,
                                      int64_t ld_t, hpfp8_stream_t stream) {
  HPFP8_REQUIRE(rows >= 0 && cols >= 0 && cols % 8 == 0 && ld % 8 == 0 && ld >= cols, HPFP8_ERR_SHAPE, "rows=%lld cols=%lld ld=%lld", (long long)rows,
                (long long)cols, (long long)ld);
  HPFP8_REQUIRE(ld_t % 8 == 0 && ld_t >= up(rows, 64), HPFP8_ERR_SHAPE, "ld_t=%lld does not hold %lld values and the zeros behind them", (long long)ld_t,
                (long long)rows);
  if (rows == 0 || cols == 0) return HPFP8_OK;
  HPFP8_REQUIRE(x && x_t, HPFP8_ERR_ARG, "null buffer");
  HPFP8_REQUIRE(aligned16(x) && aligned16(x_t), HPFP8_ERR_ALIGN, "a buffer is not 16-byte aligned");
  HPFP8_REQUIRE((cols + 63) / 64 < 65536, HPFP8_ERR_SHAPE, "too many columns");
  ce_transpose_kernel<<<dim3((unsigned)((rows + 63) / 64), (unsigned)((cols + 63) / 64)), 256, 0, (hipStream_t)stream>>>((const uint16_t*)x, ld, rows, cols, target, ignore_index,
                                                                                                                    (uint16_t*)x_t, ld_t);
  return check_launch("linear_cross_entropy_rows_t");
}

int hpfp8_linear_cross_entropy_round(const float* x, int64_t n, int parts, void* y, hpfp8_stream_t stream) {
  HPFP8_REQUIRE(parts >= 1, HPFP8_ERR_ARG, "%d parts", parts);
  HPFP8_REQUIRE(n >= 0 && n % 8 == 0, HPFP8_ERR_SHAPE, "n=%lld is no multiple of 8", (long long)n);
  if (n == 0) return HPFP8_OK;
  HPFP8_REQUIRE(x && y, HPFP8_ERR_ARG, "null buffer");
  HPFP8_REQUIRE(aligned16(x) && aligned16(y), HPFP8_ERR_ALIGN, "a buffer is not 16-byte aligned");
  ce_round_kernel<<<(unsigned)((n / 8 + 255) / 256), 256, 0, (hipStream_t)stream>>>(x, n / 8, parts, (uint16_t*)y);
  return check_launch("linear_cross_entropy_round");
}

}  // extern "C"
