// Writing new tokens' keys and values into the pages of a cache, and reading what sequences hold back, on gfx950.
//
// A cache of q's element type holds the values as they are. An e4m3 cache (8 bits: sign, 4 exponent, 3 mantissa bits,
// largest value 448) holds each row of d values of a head with one scale 2^s:
//   s = the least integer with max|x| <= 448 * 2^s (over the finite values; 0 for a row of zeros; within +-126)
//   code = x / 2^s rounded to the nearest e4m3, ties to even;  value = code * 2^s.
// A power of two makes the division and the product exact, so the rounding to e4m3 is the only one (at most 2^-4
// of a value, or 2^-10 of 2^s below 2^-6 * 2^s), and it costs e4m3 nothing: its own exponent takes up the factor of
// up to two by which the largest code may stay below 448. Values that are not finite become e4m3's NaN.
//
// What bounds both: HBM bytes, each row once in and once out. A row of one head belongs to 8, 16 or 32 lanes with 8
// values each (16-byte loads of 16-bit values, 8-byte stores of codes); keys and values go in the same thread, so
// that the page lookup, a chain of dependent loads, is paid once. 65536 tokens of 8 heads of 128, bf16: written as e4m3
// in 81 us, 5.0 TB/s (113 with 64-bit divisions, values widened one by one and non-finite ones looked for in each), read
// back in 80, and moved as they are in 100 each way, 5.3 TB/s; a copy reaches 4.8 to 5.1. A few tokens are latency: 3.3 us.
#include <type_traits>

#include "paged.hpp"

namespace samhip {

namespace {

struct KvWriteParams {
  PagedKv c;
  const void* k;
  const void* v;
  long sk[2], sv[2];
  int rows;  // tokens * heads, below 2^27
  unsigned hmagic, hshift;  // division by heads
};

struct KvReadParams {
  PagedKv c;
  void* k;
  void* v;
  int max_len;
  int rows;  // batch * max_len * heads, below 2^27
  unsigned hmagic, hshift, lmagic, lshift;  // divisions by heads and max_len
};

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

// Largest of v over a row's LPR lanes, in each 16-bit half (T of 16 bits) or as one number. Every lane calls it.
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
template <typename T, int LPR> __device__ __forceinline__ unsigned row_max(unsigned v) {
  v = larger<T>(v, moved<0xb1>(v));   // quad_perm 1 0 3 2
  v = larger<T>(v, moved<0x4e>(v));   // quad_perm 2 3 0 1
  v = larger<T>(v, moved<0x141>(v));  // mirrored in 8 lanes
  if (LPR >= 16) v = larger<T>(v, moved<0x140>(v));  // in 16
  if (LPR == 32) v = larger<T>(v, (unsigned)__shfl_xor((int)v, 16));
  return v;
}

// Largest magnitude of a lane's 8 values, as T's bits (16-bit T: in the low half).
template <typename T> __device__ __forceinline__ unsigned magnitude(const Eight<T>& x) {
  constexpr unsigned sign = sizeof(T) == 2 ? 0x7fff7fffu : 0x7fffffffu;
  unsigned top = 0;
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) top = larger<T>(top, x.w[i][j] & sign);
  return sizeof(T) == 2 ? max(top >> 16, top & 0xffffu) : top;
}
// The same over the values that are finite.
template <typename T> __device__ __forceinline__ unsigned finite_magnitude(const Eight<T>& x) {
  typedef typename std::conditional<sizeof(T) == 2, unsigned short, unsigned>::type U;
  constexpr unsigned inf = __is_same(T, f16) ? 0x7c00u : __is_same(T, bf16) ? 0x7f80u : 0x7f800000u;
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
  unsigned b;
  if constexpr (__is_same(T, f16))
    b = __float_as_uint((float)__builtin_bit_cast(f16, (unsigned short)top));
  else
    b = sizeof(T) == 2 ? top << 16 : top;
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

// Both rows' codes and scales. The maximum is taken over all bits first, the finite ones again where the result is not
// finite in some row of the wave.
template <typename T, int LPR>
__device__ __forceinline__ void quantise(const Eight<T>& k, const Eight<T>& v, u32x2& kc, u32x2& vc, int& ks, int& vs) {
  constexpr unsigned inf = __is_same(T, f16) ? 0x7c00u : __is_same(T, bf16) ? 0x7f80u : 0x7f800000u;
  unsigned kt, vt;
  auto over_rows = [&](unsigned a, unsigned b) {
    if constexpr (sizeof(T) == 2) {
      const unsigned both = row_max<T, LPR>(a | b << 16);
      kt = both & 0xffffu;
      vt = both >> 16;
    } else {
      kt = row_max<T, LPR>(a);
      vt = row_max<T, LPR>(b);
    }
  };
  over_rows(magnitude(k), magnitude(v));
  const bool odd = wave_any(kt >= inf || vt >= inf);
  if (odd) over_rows(finite_magnitude(k), finite_magnitude(v));
  ks = scale_of<T>(kt);
  vs = scale_of<T>(vt);
  kc = codes_of(k, ks, odd);
  vc = codes_of(v, vs, odd);
}

// The sequence of token t: how many sequences end at or before it. Every lane of the wave calls it; the starts come
// 64 at a time, one to a lane, and each of the wave's tokens counts over them.
template <int LPR> __device__ __forceinline__ int sequence_of(const PagedKv& c, int t) {
  const int lane = threadIdx.x & 63;
  int n = 0;
  for (int b0 = 0; b0 < c.batch; b0 += 64) {
    const int end = b0 + lane < c.batch ? c.starts[b0 + lane + 1] : 0x7fffffff;
#pragma unroll
    for (int r = 0; r < 64 / LPR; ++r) {
      const int tr = __builtin_amdgcn_readlane(t, r * LPR);
      const int ended = __popcll(__builtin_amdgcn_ballot_w64(end <= tr));
      n += lane / LPR == r ? ended : 0;
    }
  }
  return n;
}

template <typename T, bool FP8, int LPR>
__global__ __launch_bounds__(256) void kv_write_kernel(KvWriteParams p) {
  const int r = (int)((blockIdx.x * 256u + threadIdx.x) / LPR);
  const int col = (int)(threadIdx.x % LPR) * 8;
  const bool inside = r < p.rows && col < p.c.d;
  const int own = min(r, p.rows - 1), t = (int)divide_magic((unsigned)own, p.hmagic, p.hshift), head = own - t * p.c.heads;
  Eight<T> k = {}, v = {};
  if (inside) {
    k = load_eight(reinterpret_cast<const T*>(p.k) + t * p.sk[0] + head * p.sk[1] + col);
    v = load_eight(reinterpret_cast<const T*>(p.v) + t * p.sv[0] + head * p.sv[1] + col);
  }
  const int b = sequence_of<LPR>(p.c, t);
  long row = -1;  // 64 bits: row * d passes 32
  if (r < p.rows && b < p.c.batch && t >= p.c.starts[b] && t < p.c.starts[b + 1]) {
    const long j = (long)p.c.lens[b] - p.c.starts[b + 1] + t;  // its position: the last tokens of the sequence
    if (j >= 0 && j < (long)p.c.width * p.c.page) row = paged_row(p.c, b, head, (int)j, p.c.width * p.c.page);
  }
  if constexpr (FP8) {
    u32x2 kc, vc;
    int ks, vs;
    quantise<T, LPR>(k, v, kc, vc, ks, vs);
    if (row < 0 || !inside) return;
    *reinterpret_cast<u32x2*>(reinterpret_cast<unsigned char*>(p.c.k) + row * p.c.d + col) = kc;
    *reinterpret_cast<u32x2*>(reinterpret_cast<unsigned char*>(p.c.v) + row * p.c.d + col) = vc;
    if (col == 0) {
      p.c.ks[row] = (unsigned char)(ks + 127);
      p.c.vs[row] = (unsigned char)(vs + 127);
    }
  } else {
    if (row < 0 || !inside) return;
    store_eight(reinterpret_cast<T*>(p.c.k) + row * p.c.d + col, k);
    store_eight(reinterpret_cast<T*>(p.c.v) + row * p.c.d + col, v);
  }
}

// 8 codes times the row's scale as T. A value beyond T's range (an f16 one of a row written from bf16 or f32)
// rounds as the conversion does.
template <typename T> __device__ __forceinline__ Eight<T> dequantise(u32x2 c, float s) {
  typedef float f2 __attribute__((ext_vector_type(2)));
  Eight<T> r;
  T* e = reinterpret_cast<T*>(&r);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const f2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[i], false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[i], true);
    e[4 * i] = from_f32<T>(a[0] * s);
    e[4 * i + 1] = from_f32<T>(a[1] * s);
    e[4 * i + 2] = from_f32<T>(b[0] * s);
    e[4 * i + 3] = from_f32<T>(b[1] * s);
  }
  return r;
}

template <typename T, bool FP8, int LPR>
__global__ __launch_bounds__(256) void kv_read_kernel(KvReadParams p) {
  const int r = (int)((blockIdx.x * 256u + threadIdx.x) / LPR);
  const int col = (int)(threadIdx.x % LPR) * 8;
  if (r >= p.rows || col >= p.c.d) return;
  const int bj = (int)divide_magic((unsigned)r, p.hmagic, p.hshift), head = r - bj * p.c.heads;
  const int b = (int)divide_magic((unsigned)bj, p.lmagic, p.lshift), j = bj - b * p.max_len;
  const long row = paged_row(p.c, b, head, j, paged_len(p.c, b));
  Eight<T> k = {}, v = {};
  if (row >= 0) {
    if constexpr (FP8) {
      const u32x2 kc = *reinterpret_cast<const u32x2*>(reinterpret_cast<const unsigned char*>(p.c.k) + row * p.c.d + col);
      const u32x2 vc = *reinterpret_cast<const u32x2*>(reinterpret_cast<const unsigned char*>(p.c.v) + row * p.c.d + col);
      const float ks = pow2_of(p.c.ks[row]), vs = pow2_of(p.c.vs[row]);
      k = dequantise<T>(kc, ks);
      v = dequantise<T>(vc, vs);
    } else {
      k = load_eight(reinterpret_cast<const T*>(p.c.k) + row * p.c.d + col);
      v = load_eight(reinterpret_cast<const T*>(p.c.v) + row * p.c.d + col);
    }
  }
  store_eight(reinterpret_cast<T*>(p.k) + (long)r * p.c.d + col, k);
  store_eight(reinterpret_cast<T*>(p.v) + (long)r * p.c.d + col, v);
}

template <typename T, bool FP8> hipError_t write_launch(const KvWriteParams& p, hipStream_t stream) {
  const int lpr = p.c.d <= 64 ? 8 : p.c.d <= 128 ? 16 : 32;
  const dim3 grid((unsigned)(((long)p.rows * lpr + 255) / 256));
  if (lpr == 8)
    hipLaunchKernelGGL((kv_write_kernel<T, FP8, 8>), grid, dim3(256), 0, stream, p);
  else if (lpr == 16)
    hipLaunchKernelGGL((kv_write_kernel<T, FP8, 16>), grid, dim3(256), 0, stream, p);
  else
    hipLaunchKernelGGL((kv_write_kernel<T, FP8, 32>), grid, dim3(256), 0, stream, p);
  return hipGetLastError();
}

template <typename T, bool FP8> hipError_t read_launch(const KvReadParams& p, hipStream_t stream) {
  const int lpr = p.c.d <= 64 ? 8 : p.c.d <= 128 ? 16 : 32;
  const dim3 grid((unsigned)(((long)p.rows * lpr + 255) / 256));
  if (lpr == 8)
    hipLaunchKernelGGL((kv_read_kernel<T, FP8, 8>), grid, dim3(256), 0, stream, p);
  else if (lpr == 16)
    hipLaunchKernelGGL((kv_read_kernel<T, FP8, 16>), grid, dim3(256), 0, stream, p);
  else
    hipLaunchKernelGGL((kv_read_kernel<T, FP8, 32>), grid, dim3(256), 0, stream, p);
  return hipGetLastError();
}

}  // namespace

hipError_t kv_write(int dtype, int cache_dtype, const void* k, const void* v, const long* sk, const long* sv,
                    const PagedKv& c, int tokens, hipStream_t stream) {
  KvWriteParams p{c, k, v, {sk[0], sk[1]}, {sv[0], sv[1]}, tokens * c.heads, 0, 0};
  if (p.rows == 0) return hipSuccess;
  division_magic(c.heads, &p.hmagic, &p.hshift);
  if (cache_dtype == kE4M3)
    return dtype == kF32 ? write_launch<float, true>(p, stream)
                         : dtype == kF16 ? write_launch<f16, true>(p, stream) : write_launch<bf16, true>(p, stream);
  // moves of 2 or 4 bytes a value, whatever they mean
  return dtype == kF32 ? write_launch<float, false>(p, stream) : write_launch<f16, false>(p, stream);
}

hipError_t kv_read(int dtype, int cache_dtype, void* k, void* v, const PagedKv& c, int max_len, hipStream_t stream) {
  KvReadParams p{c, k, v, max_len, c.batch * max_len * c.heads, 0, 0, 0, 0};
  if (p.rows == 0) return hipSuccess;
  division_magic(c.heads, &p.hmagic, &p.hshift);
  division_magic(max_len, &p.lmagic, &p.lshift);
  if (cache_dtype == kE4M3)
    return dtype == kF32 ? read_launch<float, true>(p, stream)
                         : dtype == kF16 ? read_launch<f16, true>(p, stream) : read_launch<bf16, true>(p, stream);
  return dtype == kF32 ? read_launch<float, false>(p, stream) : read_launch<f16, false>(p, stream);
}

}  // namespace samhip
