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
// that the page lookup, a chain of dependent loads, is paid once.
#include "paged.hpp"

namespace samhip {

namespace {

struct KvWriteParams {
  PagedKv c;
  const void* k;
  const void* v;
  long sk[2], sv[2];
  int tokens;
  long rows;  // tokens * heads
};

struct KvReadParams {
  PagedKv c;
  void* k;
  void* v;
  int max_len;
  long rows;  // batch * max_len * heads
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

// The codes of this lane's 8 values, with the row's scale over its LPR lanes.
template <typename T, int LPR>
__device__ __forceinline__ u32x2 quantise(const Eight<T>& x, bool inside, unsigned char& scale) {
  const T* e = reinterpret_cast<const T*>(&x);
  float f[8];
  unsigned top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    f[i] = inside ? to_f32(e[i]) : 0.f;
    const unsigned b = __float_as_uint(f[i]) & 0x7fffffffu;
    top = max(top, b < 0x7f800000u ? b : 0u);
  }
#pragma unroll
  for (int m = 1; m < LPR; m *= 2) top = max(top, (unsigned)__shfl_xor((int)top, m, LPR));
  // max|x| = 1.f * 2^e: at most 448 * 2^s = 1.75 * 2^(8 + s)
  int s = (int)(top >> 23) - 127 - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
  s = top ? max(s, -126) : 0;
  scale = (unsigned char)(s + 127);
  const float inv = __uint_as_float((unsigned)(127 - s) << 23);
  unsigned r[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(f[4 * i] * inv, f[4 * i + 1] * inv, 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(f[4 * i + 2] * inv, f[4 * i + 3] * inv, w, true);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if ((__float_as_uint(f[4 * i + j]) & 0x7fffffffu) >= 0x7f800000u) w = (w & ~(0xff << (8 * j))) | (0x7f << (8 * j));
    r[i] = (unsigned)w;
  }
  return u32x2{r[0], r[1]};
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
  const long r = ((long)blockIdx.x * 256 + threadIdx.x) / LPR;
  const int col = (int)(threadIdx.x % LPR) * 8;
  const bool inside = r < p.rows && col < p.c.d;
  const int t = (int)(min(r, p.rows - 1) / p.c.heads), head = (int)(min(r, p.rows - 1) % p.c.heads);
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
    unsigned char ks, vs;
    const u32x2 kc = quantise<T, LPR>(k, inside, ks), vc = quantise<T, LPR>(v, inside, vs);
    if (row < 0 || !inside) return;
    *reinterpret_cast<u32x2*>(reinterpret_cast<unsigned char*>(p.c.k) + row * p.c.d + col) = kc;
    *reinterpret_cast<u32x2*>(reinterpret_cast<unsigned char*>(p.c.v) + row * p.c.d + col) = vc;
    if (col == 0) {
      p.c.ks[row] = ks;
      p.c.vs[row] = vs;
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
  const long r = ((long)blockIdx.x * 256 + threadIdx.x) / LPR;
  const int col = (int)(threadIdx.x % LPR) * 8;
  if (r >= p.rows || col >= p.c.d) return;
  const int head = (int)(r % p.c.heads);
  const long bj = r / p.c.heads;
  const int b = (int)(bj / p.max_len), j = (int)(bj % p.max_len);
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
  store_eight(reinterpret_cast<T*>(p.k) + r * p.c.d + col, k);
  store_eight(reinterpret_cast<T*>(p.v) + r * p.c.d + col, v);
}

template <typename T, bool FP8> hipError_t write_launch(const KvWriteParams& p, hipStream_t stream) {
  const int lpr = p.c.d <= 64 ? 8 : p.c.d <= 128 ? 16 : 32;
  const dim3 grid((unsigned)((p.rows * lpr + 255) / 256));
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
  const dim3 grid((unsigned)((p.rows * lpr + 255) / 256));
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
  KvWriteParams p{c, k, v, {sk[0], sk[1]}, {sv[0], sv[1]}, tokens, (long)tokens * c.heads};
  if (p.rows == 0) return hipSuccess;
  if (cache_dtype == kE4M3)
    return dtype == kF32 ? write_launch<float, true>(p, stream)
                         : dtype == kF16 ? write_launch<f16, true>(p, stream) : write_launch<bf16, true>(p, stream);
  // moves of 2 or 4 bytes a value, whatever they mean
  return dtype == kF32 ? write_launch<float, false>(p, stream) : write_launch<f16, false>(p, stream);
}

hipError_t kv_read(int dtype, int cache_dtype, void* k, void* v, const PagedKv& c, int max_len, hipStream_t stream) {
  KvReadParams p{c, k, v, max_len, (long)c.batch * max_len * c.heads};
  if (p.rows == 0) return hipSuccess;
  if (cache_dtype == kE4M3)
    return dtype == kF32 ? read_launch<float, true>(p, stream)
                         : dtype == kF16 ? read_launch<f16, true>(p, stream) : read_launch<bf16, true>(p, stream);
  return dtype == kF32 ? read_launch<float, false>(p, stream) : read_launch<f16, false>(p, stream);
}

}  // namespace samhip
