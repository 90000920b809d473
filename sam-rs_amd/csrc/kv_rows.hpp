// What the kernels that write rows of keys and values into pages share: a row's largest magnitude over its lanes, e4m3 codes
// and their scale, and the sequence that a token belongs to. A row of d values belongs to LPR lanes (8, 16 or 32) with 8 values
// each.
#pragma once
#include "paged.hpp"

namespace samhip {

// Largest of v over a row's LPR lanes, in each 16-bit half (T of 16 bits) or as one number. Every lane calls it.
template <typename T, int LPR> __device__ __forceinline__ unsigned row_max(unsigned v) {
  v = larger<T>(v, moved<0xb1>(v));   // quad_perm 1 0 3 2
  v = larger<T>(v, moved<0x4e>(v));   // quad_perm 2 3 0 1
  v = larger<T>(v, moved<0x141>(v));  // mirrored in 8 lanes
  if (LPR >= 16) v = larger<T>(v, moved<0x140>(v));  // in 16
  if (LPR == 32) v = larger<T>(v, (unsigned)__shfl_xor((int)v, 16));
  return v;
}

// The largest magnitude of a lane's 8 values, as T's bits, over those that are finite.
template <typename T> __device__ __forceinline__ unsigned finite_magnitude(const Eight<T>& x) {
  typedef typename std::conditional<sizeof(T) == 2, unsigned short, unsigned>::type U;
  constexpr unsigned inf = kInfBits<T>;
  const U* e = reinterpret_cast<const U*>(&x);
  unsigned top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const unsigned b = e[i] & (sizeof(T) == 2 ? 0x7fffu : 0x7fffffffu);
    top = max(top, b < inf ? b : 0u);
  }
  return top;
}

// The least s with top <= 448 * 2^s = 1.75 * 2^(8 + s), top = 1.f * 2^e in T's bits.
template <typename T> __device__ __forceinline__ int scale_of(unsigned top) {
  const unsigned b = f32_bits<T>(top);
  return b ? max((int)(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0), -126) : 0;
}

// The codes of two values over a power of two, in the low or the high half of w.
template <typename T, bool HI> __device__ __forceinline__ unsigned encode2(const T* e, float f, unsigned w) {
  typedef short s16x2 __attribute__((ext_vector_type(2)));
  const s16x2 old = __builtin_bit_cast(s16x2, w);
  s16x2 r;
  if constexpr (__is_same(T, f16)) {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(old, h2{e[0], e[1]}, f, HI);
  } else if constexpr (__is_same(T, bf16)) {
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(old, *reinterpret_cast<const b2*>(e), f, HI);
  } else {
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(old, e[0], e[1], f, HI);
  }
  return __builtin_bit_cast(unsigned, r);
}

// The codes of this lane's 8 values at the scale 2^s. `odd`: some lane of the wave has one that is not finite.
template <typename T> __device__ __forceinline__ u32x2 codes_of(const Eight<T>& x, int s, bool odd) {
  const T* e = reinterpret_cast<const T*>(&x);
  const float f = __uint_as_float((unsigned)(127 + s) << 23);
  unsigned r[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) r[i] = encode2<T, true>(e + 4 * i + 2, f, encode2<T, false>(e + 4 * i, f, 0u));
  if (odd) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (!(fabsf(to_f32(e[i])) < INFINITY)) r[i / 4] = (r[i / 4] & ~(0xffu << (8 * (i & 3)))) | (0x7fu << (8 * (i & 3)));
  }
  return u32x2{r[0], r[1]};
}

// One row's codes and scale: its maximum is taken over all bits first, the finite ones again where the result is not finite in
// some row of the wave. Every lane calls it.
template <typename T, int LPR> __device__ __forceinline__ void quantise_row(const Eight<T>& x, u32x2& codes, int& s) {
  unsigned top = row_max<T, LPR>(magnitude(x));
  if constexpr (sizeof(T) == 2) top &= 0xffffu;
  const bool odd = wave_any(top >= kInfBits<T>);
  if (odd) top = row_max<T, LPR>(finite_magnitude(x));
  s = scale_of<T>(top);
  codes = codes_of(x, s, odd);
}

// The sequence of token t: how many sequences end at or before it. Every lane of the wave calls it; the ends come 64 at a
// time, one to a lane (0x7fffffff past the last; the first 64 from the caller), and each of the wave's tokens counts over them.
template <int LPR> __device__ __forceinline__ int sequence_of(const PagedKv& c, int t, int end) {
  const int lane = threadIdx.x & 63;
  int n = 0;
  for (int b0 = 0;;) {
#pragma unroll
    for (int r = 0; r < 64 / LPR; ++r) {
      const int tr = __builtin_amdgcn_readlane(t, r * LPR);
      const int ended = __popcll(__builtin_amdgcn_ballot_w64(end <= tr));
      n += lane / LPR == r ? ended : 0;
    }
    b0 += 64;
    if (b0 >= c.batch) return n;
    end = b0 + lane < c.batch ? c.starts[b0 + lane + 1] : 0x7fffffff;
  }
}

}  // namespace samhip
