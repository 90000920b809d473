// Microscaled 4-bit numbers on gfx950: blocks of 32 consecutive values of a row, each value an e2m1 code (sign, 2 exponent
// bits, 1 mantissa bit: 0 0.5 1 1.5 2 3 4 6) times the block's scale, a power of two held as its biased exponent:
//   s = the least integer within +-126 with max|x| <= 6 * 2^s (0 for a block of zeros), held as s + 127
//   code = x / 2^s rounded to the nearest e2m1, ties to even;  value = code * 2^s.
// The division and the product are exact, so the rounding to e2m1 is the only one (at most a quarter of a value, and a
// quarter of 2^s below 2^s). e2m1 has no NaN: a block with a value that is not finite has the scale byte 255 and is NaN
// throughout, as the matrix units and conversions take it. Two codes share a byte, the even column's in the low half.
#pragma once
#include <type_traits>

#include "common.hpp"

namespace samhip {

constexpr int kMxBlock = 32;

// Eight consecutive values of a row, as 16-byte vectors.
template <typename T> struct Eight {
  u32x4 w[sizeof(T) / 2];
};
template <typename T> __device__ __forceinline__ Eight<T> load_eight(const T* p) {
  Eight<T> r;
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) r.w[i] = reinterpret_cast<const u32x4*>(p)[i];
  return r;
}
template <typename T> __device__ __forceinline__ void store_eight(T* p, const Eight<T>& r) {
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<u32x4*>(p)[i] = r.w[i];
}

// The larger of a and b, in each 16-bit half (T of 16 bits) or as one number.
template <typename T> __device__ __forceinline__ unsigned larger(unsigned a, unsigned b) {
  if constexpr (sizeof(T) == 2) {
    typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(unsigned, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
  } else {
    return max(a, b);
  }
}
template <int CTRL> __device__ __forceinline__ unsigned moved(unsigned v) {
  return (unsigned)__builtin_amdgcn_update_dpp((int)v, (int)v, CTRL, 0xf, 0xf, true);
}

// Largest magnitude of a lane's 8 values, as T's bits (16-bit T: in the low half). NaN is above infinity, as bits are.
template <typename T> __device__ __forceinline__ unsigned magnitude(const Eight<T>& x) {
  constexpr unsigned sign = sizeof(T) == 2 ? 0x7fff7fffu : 0x7fffffffu;
  unsigned top = 0;
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) top = larger<T>(top, x.w[i][j] & sign);
  return sizeof(T) == 2 ? max(top >> 16, top & 0xffffu) : top;
}
template <typename T> constexpr unsigned kInfBits = __is_same(T, f16) ? 0x7c00u : __is_same(T, bf16) ? 0x7f80u : 0x7f800000u;

// T's bits of a finite magnitude as f32's.
template <typename T> __device__ __forceinline__ unsigned f32_bits(unsigned top) {
  if constexpr (__is_same(T, f16))
    return __float_as_uint((float)__builtin_bit_cast(f16, (unsigned short)top));
  else
    return sizeof(T) == 2 ? top << 16 : top;
}

// The least s within +-126 with top <= 1.5 * 2^(s + 2), top = 1.f * 2^e in f32's bits.
__device__ __forceinline__ int mx_scale_of(unsigned b) {
  return b ? max((int)(b >> 23) - 127 - 2 + ((b & 0x7fffffu) > 0x400000u ? 1 : 0), -126) : 0;
}

// The codes of two values over the power of two f, as byte SEL of w.
template <typename T, int SEL> __device__ __forceinline__ unsigned mx_encode2(const T* e, float f, unsigned w) {
  if constexpr (__is_same(T, f16)) {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, h2{e[0], e[1]}, f, SEL);
  } else if constexpr (__is_same(T, bf16)) {
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, *reinterpret_cast<const b2*>(e), f, SEL);
  } else {
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, e[0], e[1], f, SEL);
  }
}

// Codes and scale byte of a lane's 8 values, whose block it shares with the other lanes of its quad. Every lane calls it.
template <typename T> __device__ __forceinline__ unsigned mx_quantise(const Eight<T>& x, unsigned& scale) {
  unsigned top = magnitude(x);
  top = max(top, moved<0xb1>(top));  // quad_perm 1 0 3 2
  top = max(top, moved<0x4e>(top));  // quad_perm 2 3 0 1
  const bool fine = top < kInfBits<T>;
  const unsigned s = (unsigned)(mx_scale_of(f32_bits<T>(fine ? top : 0u)) + 127);
  const float f = __uint_as_float(s << 23);
  const T* e = reinterpret_cast<const T*>(&x);
  const unsigned w = mx_encode2<T, 3>(e + 6, f, mx_encode2<T, 2>(e + 4, f, mx_encode2<T, 1>(e + 2, f, mx_encode2<T, 0>(e, f, 0u))));
  scale = fine ? s : 255u;
  return fine ? w : 0u;
}

// A block's scale for the conversions below, which read its exponent alone: 0 is 2^-127, 255 NaN.
__device__ __forceinline__ float mx_scale(unsigned byte) { return __uint_as_float(byte << 23); }
// Two values of a word of eight codes (byte SEL) in T, rounded to it once.
template <typename T, int SEL> __device__ __forceinline__ unsigned mx_decode2(unsigned w, float s) {
  if constexpr (__is_same(T, f16))
    return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, SEL));
  else
    return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, SEL));
}
typedef float f32x2 __attribute__((ext_vector_type(2)));
template <int SEL> __device__ __forceinline__ f32x2 mx_decode2_f32(unsigned w, float s) {
  return __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, SEL);
}
template <typename T> __device__ __forceinline__ Eight<T> mx_dequantise(unsigned w, float s) {
  Eight<T> r;
  if constexpr (sizeof(T) == 2) {
    r.w[0] = u32x4{mx_decode2<T, 0>(w, s), mx_decode2<T, 1>(w, s), mx_decode2<T, 2>(w, s), mx_decode2<T, 3>(w, s)};
  } else {
    const f32x2 a = mx_decode2_f32<0>(w, s), b = mx_decode2_f32<1>(w, s), c = mx_decode2_f32<2>(w, s), d = mx_decode2_f32<3>(w, s);
    r.w[0] = __builtin_bit_cast(u32x4, f32x4{a[0], a[1], b[0], b[1]});
    r.w[1] = __builtin_bit_cast(u32x4, f32x4{c[0], c[1], d[0], d[1]});
  }
  return r;
}

hipError_t mx_pack(int dtype, const void* x, unsigned char* codes, unsigned char* scales, long blocks, hipStream_t stream);
hipError_t mx_unpack(int dtype, const unsigned char* codes, const unsigned char* scales, void* x, long blocks, hipStream_t stream);

// out [m, n] = act(A B^T + bias), A [m, k] and B [n, k] as codes and scales, bias [n] or null. With sa null, a is A itself, in
// out's type: it is packed on the way, as mx_packs_on_the_way() calls are.
bool mx_packs_on_the_way(int m, int n, int k);
struct MxProduct {
  const void* a;
  const unsigned char* sa;
  const unsigned char* b;
  const unsigned char* sb;
  const void* bias;
  void* out;
  int m, n, k, gelu;
};
hipError_t mx_matmul(int dtype, const MxProduct& p, hipStream_t stream);

}  // namespace samhip
