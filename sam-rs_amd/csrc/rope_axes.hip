// Rotary positions over several axes (time, row, column) on gfx950: pair i of a head turns by the angle
// pos[axes[i]] * freqs[i], so that a product of two turned rows depends on the differences of their positions
// along every axis:
//   y0 = x0 cos a - x1 sin a, y1 = x1 cos a + x0 sin a
// for the pair (x[2i], x[2i+1]), or (x[i], x[i + P]) in the halves layout (P pairs); columns past 2 P are copied.
// The inverse turns by -a, which is also the gradient's way back: dL/dx is the inverse of dL/dy. The tables of
// sam_hip_rope (sam3/video.rs:106-113, rope_tables_hd, sam3/vision.rs:26-46) are the two-axis case on a fixed grid.
//
// Angles: the number of turns pos * freq / (2 pi) is formed in f64 and its fraction alone goes to f32, so that a
// position of 2^31 still has its angle to 2^-23 of a turn; sine and cosine are Taylor sums on an eighth of a turn
// either way (the first terms left out are below 2e-9 and 2e-10), exact to f32's rounding.
//
// What bounds it: HBM bytes, x once in and once out. A thread takes one 16-byte vector of a token (a pair of them in
// the halves layout), computes its angles once and turns up to 4 heads with them; its loads come before the angles.
#include "paged.hpp"

namespace samhip {

namespace {

struct RopeAxesParams {
  const void* x;
  const int* pos;
  const double* freqs;
  const int* axes;
  void* out;
  long sx[3], sp[3], so[3];
  int l, h, d, pairs, naxes;
  int halves, copy;  // copy: columns past 2 * pairs are to be written too
  int units, hgroups;  // vectors (or elements) of a head to handle, groups of heads
  long total;        // b * l * units * hgroups threads
  float sign;
};

__device__ __forceinline__ void turn_of(double freq, int pos, float sign, float& c, float& s) {
  const double t = (double)pos * (freq * 0.15915494309189533577);
  const float f = (float)(t - rint(t));       // turns, -1/2 .. 1/2
  const float k = rintf(4.f * f);
  const float y = 6.2831853071795864769f * (f - 0.25f * k), y2 = y * y;  // f - k / 4 is exact
  const float sn = y + y * y2 * (-1.f / 6 + y2 * (1.f / 120 + y2 * (-1.f / 5040 + y2 * (1.f / 362880))));
  const float cs = 1.f + y2 * (-0.5f + y2 * (1.f / 24 + y2 * (-1.f / 720 + y2 * (1.f / 40320 - y2 * (1.f / 3628800)))));
  const int q = (int)k & 3;  // quarter turns: (c, s) -> (-s, c) each
  const float a = q & 1 ? -sn : cs, b = q & 1 ? cs : sn;
  c = q & 2 ? -a : a;
  s = sign * (q & 2 ? -b : b);
}

template <typename T> struct Vec8 {
  T v[8];
};
template <typename T> __device__ __forceinline__ Vec8<T> load8(const T* p) {
  Vec8<T> r;
  u32x4* w = reinterpret_cast<u32x4*>(r.v);
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) w[i] = reinterpret_cast<const u32x4*>(p)[i];
  return r;
}
template <typename T> __device__ __forceinline__ void store8(T* p, const Vec8<T>& r) {
  const u32x4* w = reinterpret_cast<const u32x4*>(r.v);
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<u32x4*>(p)[i] = w[i];
}

template <typename T> __device__ __forceinline__ void turn(T& a, T& b, float c, float s) {
  const float x0 = to_f32(a), x1 = to_f32(b);
  a = from_f32<T>(f32_result(fmaf(x0, c, -(x1 * s))));
  b = from_f32<T>(f32_result(fmaf(x1, c, x0 * s)));
}

// Vectors of 8 elements; a thread's HP heads are hgroups apart, so that they are in flight together.
template <typename T, int HP>
__global__ __launch_bounds__(256) void rope_axes_vec(RopeAxesParams p) {
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= p.total) return;
  const int u = (int)(i % p.units);
  const long r = i / p.units;
  const int hg = (int)(r % p.hgroups);
  const long tok = r / p.hgroups;
  const long bi = tok / p.l, li = tok % p.l;
  const T* xr = reinterpret_cast<const T*>(p.x) + bi * p.sx[0] + li * p.sx[1];
  T* yr = reinterpret_cast<T*>(p.out) + bi * p.so[0] + li * p.so[1];
  const int turning = p.halves ? p.pairs / 8 : p.pairs / 4;
  const bool still = u >= turning;
  const int c0 = still ? 2 * p.pairs + 8 * (u - turning) : 8 * u;
  const int c1 = c0 + (p.halves && !still ? p.pairs : 0);  // the partners' columns
  Vec8<T> a[HP], b[HP];
#pragma unroll
  for (int k = 0; k < HP; ++k) {
    const int h = hg + k * p.hgroups;
    if (h < p.h) {
      a[k] = load8(xr + h * p.sx[2] + c0);
      if (c1 != c0) b[k] = load8(xr + h * p.sx[2] + c1);
    }
  }
  if (!still) {
    const int* pr = p.pos + bi * p.sp[0] + li * p.sp[1];
    if (p.halves) {
      float c[8], s[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int ax = p.axes[8 * u + j];
        turn_of(p.freqs[8 * u + j], (unsigned)ax < (unsigned)p.naxes ? pr[ax * p.sp[2]] : 0, p.sign, c[j], s[j]);
      }
#pragma unroll
      for (int k = 0; k < HP; ++k)
#pragma unroll
        for (int j = 0; j < 8; ++j) turn(a[k].v[j], b[k].v[j], c[j], s[j]);
    } else {
      float c[4], s[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int ax = p.axes[4 * u + j];
        turn_of(p.freqs[4 * u + j], (unsigned)ax < (unsigned)p.naxes ? pr[ax * p.sp[2]] : 0, p.sign, c[j], s[j]);
      }
#pragma unroll
      for (int k = 0; k < HP; ++k)
#pragma unroll
        for (int j = 0; j < 4; ++j) turn(a[k].v[2 * j], a[k].v[2 * j + 1], c[j], s[j]);
    }
  }
#pragma unroll
  for (int k = 0; k < HP; ++k) {
    const int h = hg + k * p.hgroups;
    if (h < p.h) {
      store8(yr + h * p.so[2] + c0, a[k]);
      if (c1 != c0) store8(yr + h * p.so[2] + c1, b[k]);
    }
  }
}

// Any sizes and strides: a thread takes one pair, or one column past the pairs, of every head of its token.
template <typename T>
__global__ __launch_bounds__(256) void rope_axes_any(RopeAxesParams p) {
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= p.total) return;
  const int u = (int)(i % p.units);
  const long tok = i / p.units;
  const long bi = tok / p.l, li = tok % p.l;
  const T* xr = reinterpret_cast<const T*>(p.x) + bi * p.sx[0] + li * p.sx[1];
  T* yr = reinterpret_cast<T*>(p.out) + bi * p.so[0] + li * p.so[1];
  if (u >= p.pairs) {
    const int col = p.pairs + u;  // 2 * pairs + (u - pairs)
    for (int h = 0; h < p.h; ++h) yr[h * p.so[2] + col] = xr[h * p.sx[2] + col];
    return;
  }
  const int c0 = p.halves ? u : 2 * u, c1 = p.halves ? u + p.pairs : 2 * u + 1, ax = p.axes[u];
  float c, s;
  turn_of(p.freqs[u], (unsigned)ax < (unsigned)p.naxes ? p.pos[bi * p.sp[0] + li * p.sp[1] + ax * p.sp[2]] : 0, p.sign,
          c, s);
  for (int h = 0; h < p.h; ++h) {
    T a = xr[h * p.sx[2] + c0], b = xr[h * p.sx[2] + c1];
    turn(a, b, c, s);
    yr[h * p.so[2] + c0] = a;
    yr[h * p.so[2] + c1] = b;
  }
}

template <typename T> hipError_t launch(RopeAxesParams p, long tokens, hipStream_t stream) {
  auto vec_ok = [](const void* q, const long* s) {
    return reinterpret_cast<uintptr_t>(q) % 16 == 0 && s[0] * (long)sizeof(T) % 16 == 0 &&
           s[1] * (long)sizeof(T) % 16 == 0 && s[2] * (long)sizeof(T) % 16 == 0;
  };
  const int rest = p.copy ? p.d - 2 * p.pairs : 0;
  const bool vec = vec_ok(p.x, p.sx) && vec_ok(p.out, p.so) && p.pairs % (p.halves ? 8 : 4) == 0 && rest % 8 == 0;
  if (!vec) {
    p.units = p.pairs + rest;
    p.hgroups = 1;
    p.total = tokens * p.units;
    hipLaunchKernelGGL(rope_axes_any<T>, dim3((unsigned)((p.total + 255) / 256)), dim3(256), 0, stream, p);
    return hipGetLastError();
  }
  p.units = p.pairs / (p.halves ? 8 : 4) + rest / 8;
  const bool four = p.h >= 4 && tokens * p.units * p.h >= 1 << 17;
  p.hgroups = four ? (p.h + 3) / 4 : p.h;
  p.total = tokens * p.units * p.hgroups;
  const dim3 grid((unsigned)((p.total + 255) / 256));
  if (four)
    hipLaunchKernelGGL((rope_axes_vec<T, 4>), grid, dim3(256), 0, stream, p);
  else
    hipLaunchKernelGGL((rope_axes_vec<T, 1>), grid, dim3(256), 0, stream, p);
  return hipGetLastError();
}

}  // namespace

hipError_t rope_axes(int dtype, const void* x, const int* pos, const double* freqs, const int* axes, void* out, int b,
                     int l, int h, int d, int pairs, int naxes, const long* sx, const long* sp, const long* so,
                     int halves, int inverse, hipStream_t stream) {
  RopeAxesParams p = {};
  p.x = x;
  p.pos = pos;
  p.freqs = freqs;
  p.axes = axes;
  p.out = out;
  for (int i = 0; i < 3; ++i) p.sx[i] = sx[i], p.sp[i] = sp[i], p.so[i] = so[i];
  p.l = l;
  p.h = h;
  p.d = d;
  p.pairs = pairs;
  p.naxes = naxes;
  p.halves = halves;
  p.copy = out != x;
  p.sign = inverse ? -1.f : 1.f;
  const long tokens = (long)b * l;
  if (tokens == 0 || (pairs == 0 && !p.copy)) return hipSuccess;
  return dtype == kF32 ? launch<float>(p, tokens, stream)
                       : dtype == kF16 ? launch<f16>(p, tokens, stream) : launch<bf16>(p, tokens, stream);
}

}  // namespace samhip
