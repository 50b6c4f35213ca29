// What the FP8 GEMM kernels share: the LDS image of an operand tile (128 bytes of one k-block per row, 16-byte chunks
// XOR-swizzled by row), fragment reads from it, bf16 packing.
#pragma once
#include "hpfp8_device.h"
#include "../../include/hpfp8.h"

namespace hpfp8 {

constexpr int BK = 128;
constexpr int kXcds = 8;             // workgroup ids congruent mod 8 share an XCD and its L2

typedef __attribute__((address_space(3))) void* lds_ptr_t;

// XOR applied to the 16-byte chunk index of tile row r.  ds_read_b128 is served 16 lanes at a time
// and the 16 are not consecutive: per half-wave the lane quads {0,3,5,6} go together and {1,2,4,7}
// go together (measured with SQ_LDS_BANK_CONFLICT on pairs of active lanes).  With the fragment
// mapping lane -> (row = lane%16, k-chunk pair = lane/16) each such group holds all 16 rows once,
// rows 4..11 with one k-chunk and the other rows with the neighbouring one; shifting the usual
// (r/2)%8 pattern by 6 sends those two row sets to disjoint chunk ranges, so the 16 lanes hit 16
// different bank groups.
__device__ __forceinline__ int row_swizzle(int r) { return (((r >> 1) & 7) + 6) & 7; }

__device__ __forceinline__ v4i lds_read16(const uint8_t* p) {
  return *reinterpret_cast<const v4i*>(p);
}

__device__ __forceinline__ v8i frag_read(const uint8_t* first, int lo_off, int hi_off) {
  v4i lo = lds_read16(first + lo_off);
  v4i hi = lds_read16(first + hi_off);
  v8i r;
  r[0] = lo[0]; r[1] = lo[1]; r[2] = lo[2]; r[3] = lo[3];
  r[4] = hi[0]; r[5] = hi[1]; r[6] = hi[2]; r[7] = hi[3];
  return r;
}
__device__ __forceinline__ v8i frag_read(const uint8_t* row_base, int pc0) { return frag_read(row_base, pc0 * 16, (pc0 ^ 1) * 16); }

// two floats -> two bf16 in one word (a low, b high): one v_cvt_pk_bf16_f32 (converted one by one, each
// value costs a conversion, a shift and an or)
__device__ __forceinline__ uint32_t pack_bf16x2(float a, float b) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, bf16x2));
}

__device__ __forceinline__ uint32_t pack_f16x2(float a, float b) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, f16x2));
}

// One k-block of int8 codes onto int32 sums (which travel in the registers of fp32 ones).  A lane's 32 bytes are two operands of the 64-wide
// instruction: each takes 16 of every lane, the same ones of both sides, so all 128 products of a row and a column are there once.
__device__ __forceinline__ v4f multiply_int8(const v8i& w, const v8i& x, const v4f& sum) {
  const v4i w0 = {w[0], w[1], w[2], w[3]}, w1 = {w[4], w[5], w[6], w[7]};
  const v4i x0 = {x[0], x[1], x[2], x[3]}, x1 = {x[4], x[5], x[6], x[7]};
  v4i s = __builtin_amdgcn_mfma_i32_16x16x64_i8(w0, x0, __builtin_bit_cast(v4i, sum), 0, 0, 0);
  s = __builtin_amdgcn_mfma_i32_16x16x64_i8(w1, x1, s, 0, 0, 0);
  return __builtin_bit_cast(v4f, s);
}

// four neighbouring values of a bias of element type HPFP8_OUT_BF16, HPFP8_OUT_F32 or HPFP8_TYPE_F16; at: a multiple of 4
__device__ __forceinline__ v4f load_bias4(const void* bias, int type, int at) {
  if (type == HPFP8_OUT_F32) return *reinterpret_cast<const v4f*>((const float*)bias + at);
  const uint2 raw = *reinterpret_cast<const uint2*>((const uint16_t*)bias + at);
  if (type == HPFP8_OUT_BF16) return v4f{bf16lo(raw.x), bf16hi(raw.x), bf16lo(raw.y), bf16hi(raw.y)};
  typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
  const f16x4 h = __builtin_bit_cast(f16x4, raw);
  return v4f{(float)h[0], (float)h[1], (float)h[2], (float)h[3]};
}

}  // namespace hpfp8
