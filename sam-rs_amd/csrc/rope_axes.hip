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

typedef int i32x4 __attribute__((ext_vector_type(4)));

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
  unsigned umagic, ushift, hmagic, hshift, lmagic, lshift;  // divisions by units, hgroups and l
  long tok0;  // this launch's first token
  int ntok;   // its tokens
  int groups;  // of a thread's tokens
  int total;  // threads: groups * hgroups * units, in this order of their digits
  float sign;
};

// Cosine and sine (times sign) of pos * freq turns.
__device__ __forceinline__ void turn_of(double freq, int pos, float sign, float& c, float& s) {
  const double t = (double)pos * freq;
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

__device__ __forceinline__ int axis_of(i32x4 v, int i) {
  const int lo = i & 1 ? v.y : v.x, hi = i & 1 ? v.w : v.z;
  return i & 2 ? hi : lo;
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

// Vectors of 8 elements: a thread takes one unit of NT tokens and HP heads of each, the tokens `groups` apart and the
// heads hgroups, so that all their loads are in flight together. The positions of up to four axes are loaded before it is
// known which of them the pairs want (AX; with more, after that).
template <typename T, int HP, int NT, bool AX>
__global__ __launch_bounds__(256) void rope_axes_vec(RopeAxesParams p) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i >= p.total) return;
  const int r = (int)divide_magic((unsigned)i, p.umagic, p.ushift), u = i - r * p.units;
  const int tg = (int)divide_magic((unsigned)r, p.hmagic, p.hshift), hg = r - tg * p.hgroups;
  const int turning = p.halves ? p.pairs / 8 : p.pairs / 4;
  const bool still = u >= turning;
  const int c0 = still ? 2 * p.pairs + 8 * (u - turning) : 8 * u;
  const int c1 = c0 + (p.halves && !still ? p.pairs : 0);  // the partners' columns
  const int first = p.halves ? 8 * u : 4 * u;              // the unit's first pair
  constexpr int NP = 8;
  Vec8<T> a[NT][HP], b[NT][HP];
  long from[NT], to[NT];
  const int* pr[NT];
  i32x4 at[NT];  // a vector: an array here, picked from by the axis, went to LDS and cost 12 us in each launch
#pragma unroll
  for (int k = 0; k < NT; ++k) {
    const long tok = p.tok0 + min(tg + (long)k * p.groups, p.ntok - 1);
    const long bi = divide_magic((unsigned)tok, p.lmagic, p.lshift), li = tok - bi * p.l;
    from[k] = bi * p.sx[0] + li * p.sx[1];
    to[k] = bi * p.so[0] + li * p.so[1];
    pr[k] = p.pos + bi * p.sp[0] + li * p.sp[1];
    if (AX) {
#pragma unroll
      for (int x = 0; x < 4; ++x) at[k][x] = pr[k][min(x, p.naxes - 1) * p.sp[2]];
    }
  }
#pragma unroll
  for (int k = 0; k < NT; ++k)
#pragma unroll
    for (int j = 0; j < HP; ++j) {
      const long h = min(hg + j * p.hgroups, p.h - 1);
      a[k][j] = load8(reinterpret_cast<const T*>(p.x) + from[k] + h * p.sx[2] + c0);
      if (c1 != c0) b[k][j] = load8(reinterpret_cast<const T*>(p.x) + from[k] + h * p.sx[2] + c1);
    }
  if (!still) {
    double f[NP];
    int ax[NP];
#pragma unroll
    for (int j = 0; j < NP; ++j)
      if (j < 4 || p.halves) {
        f[j] = p.freqs[first + j] * 0.15915494309189533577;  // turns per unit of position
        ax[j] = p.axes[first + j];
      }
#pragma unroll
    for (int k = 0; k < NT; ++k)
#pragma unroll
      for (int j = 0; j < NP; ++j)
        if (j < 4 || p.halves) {
          int x = 0;
          if ((unsigned)ax[j] < (unsigned)p.naxes) {
            if (AX)
              x = axis_of(at[k], ax[j]);
            else
              x = pr[k][ax[j] * p.sp[2]];
          }
          float c, s;
          turn_of(f[j], x, p.sign, c, s);
#pragma unroll
          for (int m = 0; m < HP; ++m) {
            if (p.halves)
              turn(a[k][m].v[j], b[k][m].v[j], c, s);
            else
              turn(a[k][m].v[2 * j & 7], a[k][m].v[(2 * j & 7) + 1], c, s);
          }
        }
  }
#pragma unroll
  for (int k = 0; k < NT; ++k)
#pragma unroll
    for (int j = 0; j < HP; ++j) {
      const int h = hg + j * p.hgroups;
      if (h < p.h && tg + (long)k * p.groups < p.ntok) {
        store8(reinterpret_cast<T*>(p.out) + to[k] + h * p.so[2] + c0, a[k][j]);
        if (c1 != c0) store8(reinterpret_cast<T*>(p.out) + to[k] + h * p.so[2] + c1, b[k][j]);
      }
    }
}

// Any sizes and strides: a thread takes one pair, or one column past the pairs, of every head of its token.
template <typename T>
__global__ __launch_bounds__(256) void rope_axes_any(RopeAxesParams p) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i >= p.total) return;
  const int t = (int)divide_magic((unsigned)i, p.umagic, p.ushift), u = i - t * p.units;
  const long tok = p.tok0 + t, bi = divide_magic((unsigned)tok, p.lmagic, p.lshift), li = tok - bi * p.l;
  const T* xr = reinterpret_cast<const T*>(p.x) + bi * p.sx[0] + li * p.sx[1];
  T* yr = reinterpret_cast<T*>(p.out) + bi * p.so[0] + li * p.so[1];
  if (u >= p.pairs) {
    const int col = p.pairs + u;  // 2 * pairs + (u - pairs)
    for (int h = 0; h < p.h; ++h) yr[h * p.so[2] + col] = xr[h * p.sx[2] + col];
    return;
  }
  const int c0 = p.halves ? u : 2 * u, c1 = p.halves ? u + p.pairs : 2 * u + 1, ax = p.axes[u];
  float c, s;
  turn_of(p.freqs[u] * 0.15915494309189533577,
          (unsigned)ax < (unsigned)p.naxes ? p.pos[bi * p.sp[0] + li * p.sp[1] + ax * p.sp[2]] : 0, p.sign, c, s);
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
  // Heads and tokens of a thread, once there are threads enough for the card. 41472 tokens of 16 heads of 64, f16: 4 and 2
  // 37.6 us, 4 and 1 43.8, 2 and 2 37.5, 2 and 4 41.7 (a copy of the bytes 34.2); f32, 65536 of 8 heads of 80: 2 and 2 62.6,
  // 4 and 2 69.0 (copy 63.4); one head of 256, 65536 tokens, bf16: 2 tokens 18.6, 4 20.7, 8 21.9, 1 25.7 (the angles; copy
  // 10.5). Halves have two vectors a head: 16384 tokens of 8 heads of 128 in f16 4 and 1 17.0, 4 and 2 18.4 (copy 14.0), one
  // head of 256 28.5 and 24.5 with 1 and 2.
  constexpr int kHeads = sizeof(T) == 4 ? 2 : 4;
  const long work = tokens * (p.d / 8) * p.h;  // vectors of 8 elements
  const int hp = vec && p.h >= 4 && work >= 1 << 17 ? kHeads : 1, nt = vec && work >= 1 << 19 && !(p.halves && hp > 1) ? 2 : 1;
  p.units = vec ? p.pairs / (p.halves ? 8 : 4) + rest / 8 : p.pairs + rest;
  p.hgroups = vec ? (p.h + hp - 1) / hp : 1;
  division_magic(p.units, &p.umagic, &p.ushift);
  division_magic(p.hgroups, &p.hmagic, &p.hshift);
  division_magic(p.l, &p.lmagic, &p.lshift);
  const long most = ((1l << 31) - 256) / ((long)p.units * p.hgroups);  // tokens of a launch: threads count in 32 bits
  for (p.tok0 = 0; p.tok0 < tokens; p.tok0 += most) {
    p.ntok = (int)(tokens - p.tok0 < most ? tokens - p.tok0 : most);
    p.groups = (p.ntok + nt - 1) / nt;
    p.total = p.groups * p.hgroups * p.units;
    const dim3 grid((unsigned)((p.total + 255l) / 256));
    auto run = [&](auto kern) { hipLaunchKernelGGL(kern, grid, dim3(256), 0, stream, p); };
    const bool ax = p.naxes <= 4 && p.pairs > 0;  // without pairs pos may be null
    if (!vec)
      run(rope_axes_any<T>);
    else if (hp > 1 && nt > 1)
      ax ? run(rope_axes_vec<T, kHeads, 2, true>) : run(rope_axes_vec<T, kHeads, 2, false>);
    else if (hp > 1)
      ax ? run(rope_axes_vec<T, kHeads, 1, true>) : run(rope_axes_vec<T, kHeads, 1, false>);
    else if (nt > 1)
      ax ? run(rope_axes_vec<T, 1, 2, true>) : run(rope_axes_vec<T, 1, 2, false>);
    else
      ax ? run(rope_axes_vec<T, 1, 1, true>) : run(rope_axes_vec<T, 1, 1, false>);
  }
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
