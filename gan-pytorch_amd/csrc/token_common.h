// What the token operators (token_rotary.hip, token_attention.hip, token_gated.hip) share: 16-byte vectors of either
// storage type and their conversion to the f32 that all arithmetic between a load and a store runs in.
#pragma once
#include "vg_internal.h"

typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

template <class T>
struct TokNum;
template <>
struct TokNum<float> {
  static constexpr int V = 4;   // elements of a 16-byte vector
};
template <>
struct TokNum<__bf16> {
  static constexpr int V = 8;
};

// a 16-byte vector as f32 (bf16 widened by a shift: exact)
__device__ __forceinline__ void tok_widen(u32x4 raw, float (&f)[4]) {
  const f32x4 v = __builtin_bit_cast(f32x4, raw);     // (of the whole vector: of an element, it reads element 0)
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = v[i];
}
__device__ __forceinline__ void tok_widen(u32x4 raw, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __builtin_bit_cast(float, raw[i] << 16);
    f[2 * i + 1] = __builtin_bit_cast(float, raw[i] & 0xffff0000u);
  }
}
// and back, each value rounded to nearest even once
__device__ __forceinline__ u32x4 tok_narrow(const float (&f)[4]) {
  u32x4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = __builtin_bit_cast(unsigned, f[i]);
  return r;
}
__device__ __forceinline__ unsigned tok_pack2(float a, float b) {
  const bf16x2 v = {(__bf16)a, (__bf16)b};
  return __builtin_bit_cast(unsigned, v);
}
__device__ __forceinline__ u32x4 tok_narrow(const float (&f)[8]) {
  u32x4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = tok_pack2(f[2 * i], f[2 * i + 1]);
  return r;
}

// Four consecutive values of either type (what a lane holds of one row of a transposed 32 x 32 product).
__device__ __forceinline__ void tok_store4(float* p, float a, float b, float c, float d) {
  *reinterpret_cast<f32x4*>(p) = f32x4{a, b, c, d};
}
__device__ __forceinline__ void tok_store4(__bf16* p, float a, float b, float c, float d) {
  *reinterpret_cast<u32x2*>(p) = u32x2{tok_pack2(a, b), tok_pack2(c, d)};
}

// Element strides of one operand; a head's elements are contiguous. Host check: every row starts on a 16-byte border.
template <class T>
static inline bool tok_layout_ok(const vg_heads_layout& l, const void* p, int64_t nb, int64_t nt, int64_t nh) {
  const int64_t V = 16 / (int64_t)sizeof(T);
  if (!vg_aligned16(p)) return false;
  return (nb <= 1 || l.sb % V == 0) && (nt <= 1 || l.st % V == 0) && (nh <= 1 || l.sh % V == 0);
}

// XCD-aware block order: workgroups are dealt to the 8 XCDs round-robin; this gives every XCD a contiguous run of the
// logical order, so that blocks that read the same operand share an L2.
__device__ __forceinline__ int tok_xcd_order(int lin, int nblk) {
  const int xcd = lin & 7, q = nblk >> 3, rem = nblk & 7;
  return (xcd < rem ? xcd * (q + 1) : rem * (q + 1) + (xcd - rem) * q) + (lin >> 3);
}
