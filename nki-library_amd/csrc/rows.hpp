// 16-byte pieces of rows of bf16, fp16 or fp32 as 32-bit values, for the operators that stream rows (token_permute.hip,
// glu_checkpoint.hip).  Rows begin wherever their length leaves them: a piece is aligned to its element only, which global
// loads and stores of any width take on this target.
#pragma once

#include "common.hpp"

namespace moe {

template <int DT>
struct Elem;
template <>
struct Elem<MOE_DT_BF16> {
  static constexpr int SIZE = 2, N = 8;
  typedef uint16_t raw;
  typedef uint32_t vec __attribute__((ext_vector_type(4), aligned(2)));
};
template <>
struct Elem<MOE_DT_FP16> {
  static constexpr int SIZE = 2, N = 8;
  typedef uint16_t raw;
  typedef uint32_t vec __attribute__((ext_vector_type(4), aligned(2)));
};
template <>
struct Elem<MOE_DT_FP32> {
  static constexpr int SIZE = 4, N = 4;
  typedef uint32_t raw;
  typedef uint32_t vec __attribute__((ext_vector_type(4), aligned(4)));
};
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef float v2f __attribute__((ext_vector_type(2)));

template <int DT>
__device__ __forceinline__ float elem_to_f32(typename Elem<DT>::raw r) {
  if constexpr (DT == MOE_DT_BF16) return bf16_bits_to_f32(r);
  else if constexpr (DT == MOE_DT_FP16) return (float)__builtin_bit_cast(_Float16, r);
  else return __uint_as_float(r);
}
template <int DT>
__device__ __forceinline__ typename Elem<DT>::raw f32_to_elem(float f) {
  if constexpr (DT == MOE_DT_BF16) return (uint16_t)pack2_bf16(f, f);
  else if constexpr (DT == MOE_DT_FP16) return __builtin_bit_cast(uint16_t, (_Float16)f);
  else return __float_as_uint(f);
}
// The 8 (4 for fp32) values of a piece.
template <int DT>
__device__ __forceinline__ void unpack(const u32x4& d, float (&v)[Elem<DT>::N]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (DT == MOE_DT_FP32) {
      v[i] = __uint_as_float(d[i]);
    } else if constexpr (DT == MOE_DT_BF16) {
      v[2 * i] = bf16_lo(d[i]);
      v[2 * i + 1] = bf16_hi(d[i]);
    } else {
      const uint32_t w = d[i];  // (a bit cast of a vector's element reads its first one)
      const v2h h = __builtin_bit_cast(v2h, w);
      v[2 * i] = (float)h[0];
      v[2 * i + 1] = (float)h[1];
    }
  }
}
template <int DT>
__device__ __forceinline__ u32x4 pack(const float (&v)[Elem<DT>::N]) {
  u32x4 d;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (DT == MOE_DT_FP32) d[i] = __float_as_uint(v[i]);
    else if constexpr (DT == MOE_DT_BF16) d[i] = pack2_bf16(v[2 * i], v[2 * i + 1]);
    else d[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector((v2f{v[2 * i], v[2 * i + 1]}), v2h));
  }
  return d;
}

// Pieces are read once and written once: past the caches' replacement order, so that what is used again stays.
template <int DT>
__device__ __forceinline__ u32x4 load_piece(const void* p) {
  const typename Elem<DT>::vec v = __builtin_nontemporal_load((const typename Elem<DT>::vec*)p);
  return u32x4{v[0], v[1], v[2], v[3]};
}
template <int DT>
__device__ __forceinline__ u32x4 load_piece_kept(const void* p) {
  const typename Elem<DT>::vec v = *(const typename Elem<DT>::vec*)p;
  return u32x4{v[0], v[1], v[2], v[3]};
}
template <int DT>
__device__ __forceinline__ void store_piece(void* p, const u32x4& d) {
  __builtin_nontemporal_store((typename Elem<DT>::vec{d[0], d[1], d[2], d[3]}), (typename Elem<DT>::vec*)p);
}

}  // namespace moe
