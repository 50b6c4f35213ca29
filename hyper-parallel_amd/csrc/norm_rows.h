// Rows of a norm: eight neighbouring values per thread and step, held in the registers of a team of 16 to 512 threads.
#pragma once
#include <type_traits>

#include "hpfp8_host.h"
#include "rows.h"

namespace hpfp8 {
namespace {

constexpr int kMaxCols = 16384;

__device__ __forceinline__ float wave_sum(float v) {
  v += __uint_as_float(dpp_u32<kDppQuadXor1>(__float_as_uint(v)));
  v += __uint_as_float(dpp_u32<kDppQuadXor2>(__float_as_uint(v)));
  v += __uint_as_float(dpp_u32<kDppRowHalfMirror>(__float_as_uint(v)));
  v += __uint_as_float(dpp_u32<kDppRowMirror>(__float_as_uint(v)));
  const int i = __builtin_bit_cast(int, v);
  auto at = [&](int lane) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(i, lane)); };
  return (at(0) + at(16)) + (at(32) + at(48));
}

// eight of w's (or b's) values as fp32; `none` where there is no such vector
__device__ __forceinline__ void load_vector8(const void* w, int type, int col, int left, float none, float v[8]) {
  if (!w) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = none;
  } else if (type == HPFP8_OUT_BF16) {
    load8<Bf16, false>((const uint16_t*)w + col, left, v);
  } else if (type == HPFP8_TYPE_F16) {
    load8<F16, false>((const _Float16*)w + col, left, v);
  } else {
    load8<F32, false>((const float*)w + col, left, v);
  }
}

// How a row's length and its chunks of eight values go together.
enum Edge {
  kWhole = 0,      // the length is a multiple of 128
  kOverlap = 1,    // any length from 8 on.  The last chunk is the row's last eight values, of which the first `dup` are the chunk's before it: every
                   // load is a whole vector, so no load has to be waited for before its turn (loads of single values of the last chunk, merged
                   // with the others' vectors, waited in every row: forward of 65536 x 1030 217 us, where this takes 86)
  kSingle = 2,     // shorter rows: value by value
};
// The chunk of eight values that a thread has in step j.
struct Chunk {
  int col;         // its first value's column
  int dup;         // values before those that are its own
  bool any;        // it has some
};
template <int EDGE>
__device__ __forceinline__ Chunk chunk_at(int index, int cols) {
  Chunk c;
  const int left = cols - index * 8;
  c.any = left > 0;
  c.dup = EDGE == kOverlap && c.any && left < 8 ? 8 - left : 0;
  c.col = c.any ? index * 8 - c.dup : 0;
  return c;
}
// whether value i of the chunk is its own
template <int EDGE>
__device__ __forceinline__ bool own(const Chunk& c, int i, int cols) {
  return EDGE == kWhole ? c.any : (EDGE == kOverlap ? c.any && i >= c.dup : c.any && c.col + i < cols);
}
template <typename E, int EDGE>
__device__ __forceinline__ Pack8<E> load_chunk(const typename E::raw* row, const Chunk& c, int cols, bool in) {
  return load_pack8<E, kStream<E>, EDGE == kSingle>(row + c.col, in && c.any ? (EDGE == kSingle ? cols - c.col : 8) : 0);
}
template <typename E, int EDGE>
__device__ __forceinline__ void store_chunk(typename E::raw* row, const Chunk& c, int cols, const float v[8]) {
  if (!c.any) return;
  if (EDGE == kWhole || (EDGE == kOverlap && c.dup == 0)) {
    store8<E, kStream<E>, false>(row + c.col, 8, v);
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (own<EDGE>(c, i, cols)) row[c.col + i] = from_f32<E>(v[i]);
}
template <int EDGE>
__device__ __forceinline__ void store_chunk_codes(uint8_t* row, const Chunk& c, int cols, uint2 codes) {
  if (!c.any) return;
  if (EDGE == kWhole || (EDGE == kOverlap && c.dup == 0)) {
    store_codes8<false>(row + c.col, 8, codes);
    return;
  }
  const uint64_t w = (uint64_t)codes.y << 32 | codes.x;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (own<EDGE>(c, i, cols)) row[c.col + i] = (uint8_t)(w >> (8 * i));
}
template <int EDGE>
__device__ __forceinline__ void vector_chunk(const void* w, int type, const Chunk& c, int cols, float none, float v[8]) {
  load_vector8(w, type, c.col, c.any ? (EDGE == kSingle ? cols - c.col : 8) : 0, none, v);
}

template <int TPR>
__device__ __forceinline__ float team_sum(float v) {          // of a wave, or of the 16 lanes of a smaller team
  if constexpr (TPR >= 64) return wave_sum(v);
  v += __uint_as_float(dpp_u32<kDppQuadXor1>(__float_as_uint(v)));
  v += __uint_as_float(dpp_u32<kDppQuadXor2>(__float_as_uint(v)));
  v += __uint_as_float(dpp_u32<kDppRowHalfMirror>(__float_as_uint(v)));
  v += __uint_as_float(dpp_u32<kDppRowMirror>(__float_as_uint(v)));
  return v;
}
template <int TPR>
__device__ __forceinline__ int team_of() {                    // (the same in a whole wave where teams are that large: a row's address is a scalar then)
  return TPR >= 64 ? __builtin_amdgcn_readfirstlane(threadIdx.x / TPR) : threadIdx.x / TPR;
}

// The smallest team that holds a row, and its steps.  f(E, threads per row, steps).  (From 1025 to 2048 values two waves of two steps are better in
// the forward, where four of one step meet at twice as many barriers, 32768 x 2048 48 / 57 us, and four in the backward, 81 / 77.)
template <typename E, bool BACKWARD, typename F>
void by_width(int cols, F&& f) {
  const int chunks = (cols + 7) / 8;
  if (chunks <= 16) f(E(), std::integral_constant<int, 16>(), std::integral_constant<int, 1>());
  else if (chunks <= 32) f(E(), std::integral_constant<int, 16>(), std::integral_constant<int, 2>());
  else if (chunks <= 64) f(E(), std::integral_constant<int, 64>(), std::integral_constant<int, 1>());
  else if (chunks <= 128) f(E(), std::integral_constant<int, 64>(), std::integral_constant<int, 2>());
  else if (chunks <= 256) f(E(), std::integral_constant<int, BACKWARD ? 256 : 128>(), std::integral_constant<int, BACKWARD ? 1 : 2>());
  else if (chunks <= 512) f(E(), std::integral_constant<int, 256>(), std::integral_constant<int, 2>());
  else if (chunks <= 1024) f(E(), std::integral_constant<int, 512>(), std::integral_constant<int, 2>());
  else f(E(), std::integral_constant<int, 512>(), std::integral_constant<int, 4>());
}
template <bool BACKWARD, typename F>
void by_type_and_width(int dtype, int cols, F&& f) {
  if (dtype == HPFP8_OUT_BF16) by_width<Bf16, BACKWARD>(cols, f);
  else if (dtype == HPFP8_TYPE_F16) by_width<F16, BACKWARD>(cols, f);
  else by_width<F32, BACKWARD>(cols, f);
}
inline bool at_element(const void* p, int dtype) { return ((uintptr_t)p & (dtype == HPFP8_OUT_F32 ? 3 : 1)) == 0; }

}  // namespace
}  // namespace hpfp8
