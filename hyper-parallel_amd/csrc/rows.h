// Eight neighbouring values of a row at a time, in any of the three element types, from any address that is a multiple of the
// element's size; and the E4M3 form of a group of 128 values, which is 16 lanes' eight values each.
#pragma once
#include "hpfp8_device.h"

namespace hpfp8 {

struct Bf16 {
  using raw = uint16_t;
};
struct F16 {
  using raw = _Float16;
};
struct F32 {
  using raw = float;
};

// Vectors that start at any element: global memory is read and written in whole vectors at such addresses too (at most one more
// cache line per wave), so rows of odd length need no kernel of their own.
typedef uint32_t u32x4_at2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x4_at4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x2_at1 __attribute__((ext_vector_type(2), aligned(1)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));

template <typename E>
__device__ __forceinline__ float to_f32(typename E::raw v) {
  if constexpr (__is_same(E, Bf16)) return __uint_as_float((uint32_t)v << 16);
  else return (float)v;
}
template <typename E>
__device__ __forceinline__ typename E::raw from_f32(float v) {
  if constexpr (__is_same(E, Bf16)) return __builtin_bit_cast(uint16_t, (__bf16)v);
  else return (typename E::raw)v;
}

// Eight values as they lie in memory: 16 bytes, or 32 of F32.
template <typename E>
struct Pack8 {
  u32x4 w[sizeof(typename E::raw) == 4 ? 2 : 1];
};

template <typename E>
__device__ __forceinline__ void unpack8(const Pack8<E>& p, float v[8]) {
  if constexpr (__is_same(E, Bf16)) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = bf16lo(p.w[0][i]);
      v[2 * i + 1] = bf16hi(p.w[0][i]);
    }
  } else if constexpr (__is_same(E, F16)) {
    const f16x8 h = __builtin_bit_cast(f16x8, p.w[0]);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)h[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(p.w[i / 4][i % 4]);
  }
}

template <typename E>
__device__ __forceinline__ Pack8<E> pack8(const float v[8]) {
  Pack8<E> p;
  if constexpr (__is_same(E, Bf16)) {
#pragma unroll
    for (int i = 0; i < 4; ++i) p.w[0][i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2_t{v[2 * i], v[2 * i + 1]}, bf16x2_t));
  } else if constexpr (__is_same(E, F16)) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float a = v[2 * i], b = v[2 * i + 1];
      // (rounded to fp32 first in every kernel: the compiler folds the conversion into a fused multiply-add in some and not in others)
      asm("" : "+v"(a), "+v"(b));
      p.w[0][i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2_t{a, b}, f16x2_t));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) p.w[i / 4][i % 4] = __float_as_uint(v[i]);
  }
  return p;
}

// Values of 16 bits are accessed as data used once.  Those of 32 are not: a lane's eight are two vectors, so each access leaves half of a cache
// line for the next one (8192 x 8192, silu with its codes 121 / 110 us, read back from codes 105 / 70).
template <typename E>
constexpr bool kStream = sizeof(typename E::raw) == 2;

// n: how many of the eight there are (8 or more: all of them; 0 or less: none); those that are not there are zeros.
// TAIL = false: all or none (a row's length is a multiple of eight).
template <typename E, bool NT = kStream<E>, bool TAIL = true>
__device__ __forceinline__ Pack8<E> load_pack8(const typename E::raw* p, int n) {
  Pack8<E> r;
  if (n >= 8) {
    if constexpr (sizeof(typename E::raw) == 4) {
      const u32x4_at4* q = reinterpret_cast<const u32x4_at4*>(p);
      r.w[0] = NT ? __builtin_nontemporal_load(q) : q[0];
      r.w[1] = NT ? __builtin_nontemporal_load(q + 1) : q[1];
    } else {
      const u32x4_at2* q = reinterpret_cast<const u32x4_at2*>(p);
      r.w[0] = NT ? __builtin_nontemporal_load(q) : q[0];
    }
    return r;
  }
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = TAIL && i < n ? to_f32<E>(p[i]) : 0.f;
  return pack8<E>(v);                      // (a value that came from E goes back to the same bits)
}
template <typename E, bool NT = kStream<E>>
__device__ __forceinline__ void load8(const typename E::raw* p, int n, float v[8]) {
  unpack8<E>(load_pack8<E, NT>(p, n), v);
}

template <typename E, bool NT = kStream<E>, bool TAIL = true>
__device__ __forceinline__ void store8(typename E::raw* p, int n, const float v[8]) {
  if (n >= 8) {
    const Pack8<E> r = pack8<E>(v);
    if constexpr (sizeof(typename E::raw) == 4) {
      u32x4_at4* q = reinterpret_cast<u32x4_at4*>(p);
      if (NT) {
        __builtin_nontemporal_store((u32x4_at4)r.w[0], q);
        __builtin_nontemporal_store((u32x4_at4)r.w[1], q + 1);
      } else {
        q[0] = r.w[0];
        q[1] = r.w[1];
      }
    } else {
      u32x4_at2* q = reinterpret_cast<u32x4_at2*>(p);
      if (NT) __builtin_nontemporal_store((u32x4_at2)r.w[0], q);
      else q[0] = r.w[0];
    }
    return;
  }
  if (!TAIL) return;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < n) p[i] = from_f32<E>(v[i]);
}

// ---- eight E4M3 codes
template <bool TAIL = true>
__device__ __forceinline__ uint2 load_codes8(const uint8_t* p, int n) {
  if (n >= 8) {
    const u32x2 v = __builtin_nontemporal_load(reinterpret_cast<const u32x2_at1*>(p));
    return make_uint2(v.x, v.y);
  }
  uint64_t w = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (TAIL && i < n) w |= (uint64_t)p[i] << (8 * i);
  return make_uint2((uint32_t)w, (uint32_t)(w >> 32));
}
template <bool TAIL = true>
__device__ __forceinline__ void store_codes8(uint8_t* p, int n, uint2 c) {
  if (n >= 8) {
    __builtin_nontemporal_store(u32x2_at1{c.x, c.y}, reinterpret_cast<u32x2_at1*>(p));
    return;
  }
  if (!TAIL) return;
  const uint64_t w = (uint64_t)c.y << 32 | c.x;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < n) p[i] = (uint8_t)(w >> (8 * i));
}

// E4M3 has one code of each sign for what is no number.  Where infinities have to come back as they were, those two are +inf and -inf,
// and NaN is the code of -0 (a value that rounds to -0 gets the code of 0).
constexpr uint32_t kCodeInf = 0x7F, kCodeNan = 0x80;
__device__ __forceinline__ uint32_t no_negative_zero(uint32_t w) {         // (a byte's upper bit stays where its others are not all 0)
  return w & (0x7F7F7F7Fu | ((w & 0x7F7F7F7Fu) + 0x7F7F7F7Fu));
}

// The group's 16 lanes' eight values each -> their codes; scale_inv is the same in all 16.  |v| orders like its bits, and a NaN
// above everything: the group's scale and codes are NaN then.  (No clamp: |v * (448 / amax)| <= 448 (1 + 2^-23), which rounds to 448.)
// SPECIAL: infinities and NaN have codes of their own, and the scale is that of the finite values.
template <bool SPECIAL = false>
__device__ __forceinline__ uint2 encode_group(const float v[8], float& scale_inv) {
  // (the maximum that keeps NaN: one instruction for two values more)
  float top = __builtin_elementwise_maximum(__builtin_fabsf(v[0]), __builtin_fabsf(v[1]));
#pragma unroll
  for (int i = 2; i < 8; i += 2) top = __builtin_elementwise_maximum(__builtin_elementwise_maximum(top, __builtin_fabsf(v[i])), __builtin_fabsf(v[i + 1]));
  const bool special = SPECIAL && !(top < INFINITY);                        // (few lanes take this way)
  if (special) {
    top = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = __builtin_fabsf(v[i]) < INFINITY ? fmaxf(top, __builtin_fabsf(v[i])) : top;
  }
  const uint32_t m = row16_max_u32(__float_as_uint(top) & 0x7FFFFFFFu);
  float scale;
  scales_from_amax(__uint_as_float(m), scale, scale_inv);
  uint2 c;
  int lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[0] * scale, v[1] * scale, 0, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[2] * scale, v[3] * scale, lo, true);
  int hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[4] * scale, v[5] * scale, 0, false);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[6] * scale, v[7] * scale, hi, true);
  c.x = (uint32_t)lo;
  c.y = (uint32_t)hi;
  if constexpr (SPECIAL) {
    c.x = no_negative_zero(c.x);
    c.y = no_negative_zero(c.y);
    if (special) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (__builtin_fabsf(v[i]) < INFINITY) continue;
        const uint32_t code = v[i] != v[i] ? kCodeNan : (v[i] < 0.f ? kCodeInf | 0x80u : kCodeInf);
        uint32_t& w = i < 4 ? c.x : c.y;
        w = (w & ~(0xFFu << 8 * (i % 4))) | code << 8 * (i % 4);
      }
    }
  }
  return c;
}
template <bool SPECIAL = false>
__device__ __forceinline__ void decode8(uint2 c, float scale_inv, float v[8]) {
  const v2f a = __builtin_amdgcn_cvt_pk_f32_fp8((int)c.x, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)c.x, true);
  const v2f d = __builtin_amdgcn_cvt_pk_f32_fp8((int)c.y, false), e = __builtin_amdgcn_cvt_pk_f32_fp8((int)c.y, true);
  v[0] = a.x * scale_inv;
  v[1] = a.y * scale_inv;
  v[2] = b.x * scale_inv;
  v[3] = b.y * scale_inv;
  v[4] = d.x * scale_inv;
  v[5] = d.y * scale_inv;
  v[6] = e.x * scale_inv;
  v[7] = e.y * scale_inv;
  if constexpr (SPECIAL) {
    // a byte whose low seven bits are all 1 is an infinity; one that no_negative_zero changes is a NaN
    const uint32_t inf = (((c.x & 0x7F7F7F7Fu) + 0x01010101u) | ((c.y & 0x7F7F7F7Fu) + 0x01010101u)) & 0x80808080u;
    if (inf || no_negative_zero(c.x) != c.x || no_negative_zero(c.y) != c.y) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t code = (i < 4 ? c.x : c.y) >> 8 * (i % 4) & 0xFFu;
        if ((code & 0x7Fu) == kCodeInf) v[i] = code & 0x80u ? -INFINITY : INFINITY;
        if (code == kCodeNan) v[i] = NAN;
      }
    }
  }
}

}  // namespace hpfp8
