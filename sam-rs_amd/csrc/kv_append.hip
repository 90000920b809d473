// New tokens into a paged cache with the position rotation on the way, on gfx950: queries and keys turn as in rope_axes.hip
//   y0 = x0 cos a - x1 sin a, y1 = x1 cos a + x0 sin a, a = pos[axes[i]] * freqs[i]
// and queries go out, keys and values into their pages as in kv_cache.hip, in one launch in place of three and without
// the turned keys' way through memory.
//
// Keys are turned in f64 and rounded once, to their type or to their codes, so that a code is the definition's also next to
// the border between two (an f32 turn, off by 2^-22, would flip one of a million). The angle is the f64 product; it is reduced
// by quarter turns with pi / 2 in two parts (exact to 2^-52 up to 2^48 radians), sine and cosine are Taylor sums on an eighth
// of a turn either way, whose first terms left out are below 2^-56. Queries, which go out in their own type, take sine
// and cosine in f32, from the angle so reduced.
//
// What bounds it: HBM bytes, each row in and out once. A row belongs to LPR lanes of 8 columns, as in kv_cache.hip; they form
// their angles once for HP heads of a token. In the halves layout a lane loads its partners' columns too (their lines are on
// their way for the partner lane), so that nothing passes between lanes and a row may be turned in place: its loads come
// before its wave's stores. Key heads come first in the grid, whose chain of table reads is the longer one.
//
// Measured: 65536 tokens of 8 query and 8 key heads of 128 in bf16, all pairs turned, into pages of bf16, e4m3 and e2m1 147,
// 130 and 117 us (5.5, 5.2 and 5.2 TB/s; kv_write of the same keys alone takes 96, 83 and 75, rope_axes of the queries 44 and of
// the keys as much again). 32 tokens of 32 and 8 heads are latency: 5.8 us, most of it the chain from the table to a store.
#include <algorithm>

#include "kv_rows.hpp"

namespace samhip {

static int lanes_of_row(int d) { return d <= 64 ? 8 : d <= 128 ? 16 : 32; }

// How many heads of a token a thread takes, which share its angles: several where there are threads enough for all CUs without,
// and as many query or key heads (the other part's threads then do less than they could, and there are fewer of them). 16 query
// heads of 128 in bf16 over 1, 2, 3 and 4 key heads, 16384 tokens: 62, 63, 66 and 71 us with one, 36, 34, 35 and 36 with four; 1024
// tokens over 1 key head 7.7 and 7.6, 512, which take one, 6.0 and 7.0; 4 over 2, 16384 tokens, 27 and 20; 2 over 2, which take one,
// 22 and 20, 1 over 1 head of 256 22 and 30. In f32, whose rows take twice the registers, two: 16 over 1, 2, 3 and 4 74, 81, 89
// and 98 with one, 64, 69, 78 and 82 with two; 512 tokens over 1, which take one, 6.1 and 5.8.
int kv_append_heads(int element, int tokens, int heads, int kv_heads, int d) {
  const long rows = (long)tokens * (heads + kv_heads);
  const int most = element == 4 ? 2 : 4;
  return rows * lanes_of_row(d) >= 1 << 18 && std::max(heads, kv_heads) >= most ? most : 1;
}

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));

struct KvAppendParams {
  PagedKv c;
  const void* q;
  const void* k;
  const void* v;
  const int* pos;  // null: a token's position in its sequence, on every axis
  const double* freqs;
  const int* axes;
  void* out;
  long sq[2], sk[2], sv[2], sp[2], so[2];
  int tokens, heads, pairs, naxes;
  int zero_rest;
  int kgroups, qgroups;                       // groups of HP heads of a token
  unsigned kmagic, kshift, qmagic, qshift;    // divisions by them
  int kunits, qunits;                         // tokens * groups
  unsigned kblocks;                           // workgroups for keys and values; the queries' follow
};

// a less the nearest k quarter turns.
__device__ __forceinline__ double reduced(double a, double& k) {
  k = rint(a * 0.63661977236758134308);
  // pi / 2 as a double, whose product with k fma takes exactly, and what it lacks
  return fma(-k, 6.12323399573676588613e-17, fma(-k, 1.57079632679489661923, a));
}
// (c, s) after k quarter turns: (c, s) -> (-s, c) each.
template <typename F> __device__ __forceinline__ void quarters(double k, F& c, F& s) {
  const int quarter = (int)(long)k & 3;
  const F u = quarter & 1 ? -s : c, w = quarter & 1 ? c : s;
  c = quarter & 2 ? -u : u;
  s = quarter & 2 ? -w : w;
}

// cos and sin of a.
__device__ __forceinline__ void turn_of(double a, double& c, double& s) {
  double k;
  const double r = reduced(a, k);
  const double r2 = r * r;
  double sn = 1.0 / 355687428096000.0, cs = -1.0 / 6402373705728000.0;  // 1 / 17!, -1 / 18!
  sn = fma(sn, r2, -1.0 / 1307674368000.0);
  cs = fma(cs, r2, 1.0 / 20922789888000.0);
  sn = fma(sn, r2, 1.0 / 6227020800.0);
  cs = fma(cs, r2, -1.0 / 87178291200.0);
  sn = fma(sn, r2, -1.0 / 39916800.0);
  cs = fma(cs, r2, 1.0 / 479001600.0);
  sn = fma(sn, r2, 1.0 / 362880.0);
  cs = fma(cs, r2, -1.0 / 3628800.0);
  sn = fma(sn, r2, -1.0 / 5040.0);
  cs = fma(cs, r2, 1.0 / 40320.0);
  sn = fma(sn, r2, 1.0 / 120.0);
  cs = fma(cs, r2, -1.0 / 720.0);
  sn = fma(sn, r2, -1.0 / 6.0);
  cs = fma(cs, r2, 1.0 / 24.0);
  sn = fma(sn * r2, r, r);
  cs = fma(cs, r2, -0.5);
  cs = fma(cs, r2, 1.0);
  c = cs;
  s = sn;
  quarters(k, c, s);
}
__device__ __forceinline__ void turn_of(double a, float& c, float& s) {
  double k;
  const float y = (float)reduced(a, k), y2 = y * y;
  s = y + y * y2 * (-1.f / 6 + y2 * (1.f / 120 + y2 * (-1.f / 5040 + y2 * (1.f / 362880))));
  c = 1.f + y2 * (-0.5f + y2 * (1.f / 24 + y2 * (-1.f / 720 + y2 * (1.f / 40320 - y2 * (1.f / 3628800)))));
  quarters(k, c, s);
}

// x in f32, rounded to odd: cut short, and its last bit set if anything was cut off. Rounding that to fewer bits (up to 22)
// gives what rounding x to them would. x beyond f32's largest number is infinite, as it is to kv_write.
__device__ __forceinline__ float to_odd(double x) {
  const float f = (float)x;
  unsigned u = __float_as_uint(f);
  if ((double)f != x && fabsf(f) < INFINITY) u = (fabs((double)f) > fabs(x) ? u - 1 : u) | 1u;
  return __uint_as_float(u);
}

// 8 values turned by their pairs' (c, s): with HALVES, x's partners are o's and `low` says which of the two x are; else pairs
// are neighbours, and a pair's (c, s) is at its first element's half.
template <typename F, bool HALVES> __device__ __forceinline__ F turned(int j, const F* x, const F* o, const F* c, const F* s, bool low) {
  if constexpr (HALVES) {
    return low ? fma(x[j], c[j], -(o[j] * s[j])) : fma(x[j], c[j], o[j] * s[j]);
  } else {
    const int i = j / 2;
    return j % 2 == 0 ? fma(x[j], c[i], -(x[j + 1] * s[i])) : fma(x[j], c[i], x[j - 1] * s[i]);
  }
}

template <typename T, typename C, int LPR, int HP, bool HALVES>
__global__ __launch_bounds__(256) void kv_append_kernel(KvAppendParams p) {
  constexpr int NP = HALVES ? 8 : 4;  // pairs of a lane
  const bool keys = blockIdx.x < p.kblocks;
  const int r = (int)(((blockIdx.x - (keys ? 0u : p.kblocks)) * 256u + threadIdx.x) / LPR);
  const int col = (int)(threadIdx.x % LPR) * 8, d = p.c.d;
  const int units = keys ? p.kunits : p.qunits, groups = keys ? p.kgroups : p.qgroups, heads = keys ? p.c.heads : p.heads;
  const int own = min(r, units - 1);
  const int t = (int)divide_magic((unsigned)own, keys ? p.kmagic : p.qmagic, keys ? p.kshift : p.qshift), hg = own - t * groups;
  const bool inside = r < units && col < d;
  // which of the lane's elements turn, and where their partners are
  unsigned turn = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) turn |= col + j < 2 * p.pairs ? 1u << j : 0u;
  // halves: a lane's elements have one role, and its partners are one load. With other counts of pairs they are loaded one by one:
  // 16384 tokens of 16 and 4 heads of 128, bf16 with 64, 48 and 32 pairs 36 us, with 45, 29 and 13 47, 51 and 55, f32 83 and 103 to
  // 109, 32 tokens 5.3 and 5.7
  const bool even = p.pairs % 8 == 0;
  const bool low = col < p.pairs;

  // Everything that depends on nothing goes out at once, the ends and lengths of the first 64 sequences first, one to a lane:
  // the way from them to the pages is the longest
  const int lane = threadIdx.x & 63;
  const int seq = min(lane, p.c.batch - 1), ends = p.c.starts[seq + 1], held = p.c.lens[seq], first = p.c.starts[0];
  Eight<T> x[HP], o[HALVES ? HP : 1], v[HP];
  auto load_rows = [&](const void* base, const long* st, Eight<T>* a, bool partners) {
#pragma unroll
    for (int i = 0; i < HP; ++i) {
      const T* row = reinterpret_cast<const T*>(base) + t * st[0] + min(hg + i * groups, heads - 1) * st[1];
      a[i] = load_eight(row + min(col, d - 8));
      if constexpr (HALVES) {
        if (!partners) continue;
        if (p.pairs == 0) {
          o[i] = Eight<T>{};
        } else if (even) {
          o[i] = load_eight(row + min(turn ? (low ? col + p.pairs : col - p.pairs) : col, d - 8));
        } else {
          T* e = reinterpret_cast<T*>(&o[i]);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int at = col + j < p.pairs ? col + j + p.pairs : col + j < 2 * p.pairs ? col + j - p.pairs : col + j;
            e[j] = row[min(at, d - 1)];
          }
        }
      }
    }
  };
  load_rows(keys ? p.k : p.q, keys ? p.sk : p.sq, x, true);
  if (keys) load_rows(p.v, p.sv, v, false);
  double freq[NP];
  int axis[NP];
  i32x4 ps = {};  // up to four axes' positions, loaded before it is known which of them the pairs want
  const int* pr = p.pos + (long)t * p.sp[0];
  if (p.pairs > 0) {
#pragma unroll
    for (int j = 0; j < NP; ++j) {
      int i = HALVES ? col + j : col / 2 + j;
      if (HALVES && i >= p.pairs) i -= p.pairs;
      i = min(i, p.pairs - 1);
      freq[j] = p.freqs[i];
      axis[j] = p.pos ? p.axes[i] : 0;
    }
    if (p.pos && p.naxes <= 4) {
#pragma unroll
      for (int a = 0; a < 4; ++a) ps[a] = pr[min(a, p.naxes - 1) * p.sp[1]];
    }
  }

  // the token's sequence and position
  const int b = sequence_of<LPR>(p.c, t, lane < p.c.batch ? ends : 0x7fffffff);
  int from, to, len;
  if (p.c.batch <= 64) {
    const int before = __shfl(ends, max(min(b, p.c.batch) - 1, 0));  // by every lane: a lane left out would give 0
    from = b > 0 ? before : first;
    to = __shfl(ends, min(b, p.c.batch - 1));
    len = __shfl(held, min(b, p.c.batch - 1));
  } else {
    const int at = min(b, p.c.batch - 1);
    from = p.c.starts[at], to = p.c.starts[at + 1], len = p.c.lens[at];
  }
  const bool known = b < p.c.batch && t >= from && t < to;
  const long at = known ? (long)len - to + t : 0;
  const long end = (long)p.c.width * p.c.page;
  const bool fits = keys && r < units && known && at >= 0 && at < end;
  PagedEntry entry = {-1, -1};
  if (fits) entry = paged_entry(p.c, b, (int)at, (int)end);

  auto angle = [&](int j) {
    if (!p.pos) return (double)at * freq[j];
    int w = 0;
    if ((unsigned)axis[j] < (unsigned)p.naxes) {
      if (p.naxes <= 4) {
        const int lo = axis[j] & 1 ? ps.y : ps.x, hi = axis[j] & 1 ? ps.w : ps.z;
        w = axis[j] & 2 ? hi : lo;
      } else {
        w = pr[axis[j] * p.sp[1]];
      }
    }
    return (double)w * freq[j];
  };

  if (!keys) {
    const bool rest = !known;
    if (!inside || (rest && !p.zero_rest)) return;
    float c[NP], s[NP];
#pragma unroll
    for (int j = 0; j < NP; ++j) {
      c[j] = 1.f, s[j] = 0.f;
      if (p.pairs > 0) turn_of(angle(j), c[j], s[j]);
    }
#pragma unroll
    for (int i = 0; i < HP; ++i) {
      const int h = hg + i * groups;
      if (h >= heads) break;
      const T* e = reinterpret_cast<const T*>(&x[i]);
      const T* po = reinterpret_cast<const T*>(&o[HALVES ? i : 0]);
      float xf[8], of[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) xf[j] = to_f32(e[j]), of[j] = HALVES ? to_f32(po[j]) : 0.f;
      Eight<T> y;
      T* ye = reinterpret_cast<T*>(&y);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float z = turned<float, HALVES>(j, xf, of, c, s, col + j < p.pairs);
        ye[j] = rest ? from_f32<T>(0.f) : turn >> j & 1 ? from_f32<T>(f32_result(z)) : e[j];
      }
      store_eight(reinterpret_cast<T*>(p.out) + t * p.so[0] + h * p.so[1] + col, y);
    }
    return;
  }

  double c[NP], s[NP];
#pragma unroll
  for (int j = 0; j < NP; ++j) {
    c[j] = 1.0, s[j] = 0.0;
    if (p.pairs > 0) turn_of(angle(j), c[j], s[j]);
  }
#pragma unroll
  for (int i = 0; i < HP; ++i) {
    const int h = hg + i * groups;
    const long row = fits && h < heads ? paged_row(p.c, entry, h) : -1;  // 64 bits: row * d passes 32
    const T* e = reinterpret_cast<const T*>(&x[i]);
    const T* po = reinterpret_cast<const T*>(&o[HALVES ? i : 0]);
    double xd[8], od[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) xd[j] = to_f32(e[j]), od[j] = HALVES ? to_f32(po[j]) : 0.f;
    constexpr bool kHeld = !__is_same(C, e4m3) && !__is_same(C, e2m1);
    Eight<float> y;
    float* ye = reinterpret_cast<float*>(&y);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const double z = turned<double, HALVES>(j, xd, od, c, s, col + j < p.pairs);
      ye[j] = turn >> j & 1 ? kHeld && sizeof(T) == 4 ? (float)z : to_odd(z) : to_f32(e[j]);
    }
    if (!inside) {  // columns past d take part in the row's maximum
      y = Eight<float>{};
      v[i] = Eight<T>{};
    }
    const long place = row * d + col;
    if constexpr (__is_same(C, e2m1)) {
      unsigned ks, vs;
      const unsigned kc = mx_quantise(y, ks), vc = mx_quantise(v[i], vs);
      if (row >= 0 && inside) {
        reinterpret_cast<unsigned*>(p.c.k)[place / 8] = kc;
        reinterpret_cast<unsigned*>(p.c.v)[place / 8] = vc;
        if (col % kMxBlock == 0) {
          p.c.ks[place / kMxBlock] = (unsigned char)ks;
          p.c.vs[place / kMxBlock] = (unsigned char)vs;
        }
      }
    } else if constexpr (__is_same(C, e4m3)) {
      u32x2 kc, vc;
      int ks, vs;
      quantise_row<float, LPR>(y, kc, ks);
      quantise_row<T, LPR>(v[i], vc, vs);
      if (row >= 0 && inside) {
        *reinterpret_cast<u32x2*>(reinterpret_cast<unsigned char*>(p.c.k) + place) = kc;
        *reinterpret_cast<u32x2*>(reinterpret_cast<unsigned char*>(p.c.v) + place) = vc;
        if (col == 0) {
          p.c.ks[row] = (unsigned char)(ks + 127);
          p.c.vs[row] = (unsigned char)(vs + 127);
        }
      }
    } else if (row >= 0 && inside) {
      Eight<T> held;
      T* he = reinterpret_cast<T*>(&held);
#pragma unroll
      for (int j = 0; j < 8; ++j) he[j] = from_f32<T>(ye[j]);
      store_eight(reinterpret_cast<T*>(p.c.k) + place, held);
      store_eight(reinterpret_cast<T*>(p.c.v) + place, v[i]);
    }
  }
}

template <typename T, typename C, int LPR, int HP> hipError_t launch(KvAppendParams p, bool halves, hipStream_t stream) {
  p.kgroups = (p.c.heads + HP - 1) / HP;
  p.qgroups = (p.heads + HP - 1) / HP;
  division_magic(p.kgroups, &p.kmagic, &p.kshift);
  if (p.qgroups) division_magic(p.qgroups, &p.qmagic, &p.qshift);
  p.kunits = p.tokens * p.kgroups;
  p.qunits = p.tokens * p.qgroups;
  p.kblocks = (unsigned)(((long)p.kunits * LPR + 255) / 256);
  const dim3 grid(p.kblocks + (unsigned)(((long)p.qunits * LPR + 255) / 256));
  if (halves)
    hipLaunchKernelGGL((kv_append_kernel<T, C, LPR, HP, true>), grid, dim3(256), 0, stream, p);
  else
    hipLaunchKernelGGL((kv_append_kernel<T, C, LPR, HP, false>), grid, dim3(256), 0, stream, p);
  return hipGetLastError();
}
template <typename T, typename C, int LPR> hipError_t by_heads(const KvAppendParams& p, bool halves, hipStream_t stream) {
  constexpr int kHeads = sizeof(T) == 4 ? 2 : 4;
  return kv_append_heads(sizeof(T), p.tokens, p.heads, p.c.heads, p.c.d) > 1 ? launch<T, C, LPR, kHeads>(p, halves, stream)
                                                                             : launch<T, C, LPR, 1>(p, halves, stream);
}
template <typename T, typename C> hipError_t by_size(const KvAppendParams& p, bool halves, hipStream_t stream) {
  const int lpr = lanes_of_row(p.c.d);
  return lpr == 8 ? by_heads<T, C, 8>(p, halves, stream) : lpr == 16 ? by_heads<T, C, 16>(p, halves, stream) : by_heads<T, C, 32>(p, halves, stream);
}
template <typename T> hipError_t by_held(int cache_dtype, const KvAppendParams& p, bool halves, hipStream_t stream) {
  return cache_dtype == kE2M1 ? by_size<T, e2m1>(p, halves, stream)
                              : cache_dtype == kE4M3 ? by_size<T, e4m3>(p, halves, stream) : by_size<T, T>(p, halves, stream);
}

}  // namespace

hipError_t kv_append(int dtype, int cache_dtype, const KvAppendCall& a, const PagedKv& c, hipStream_t stream) {
  KvAppendParams p = {};
  p.c = c;
  p.q = a.q;
  p.k = a.k;
  p.v = a.v;
  p.pos = a.pos;
  p.freqs = a.freqs;
  p.axes = a.axes;
  p.out = a.out;
  for (int i = 0; i < 2; ++i) p.sq[i] = a.sq[i], p.sk[i] = a.sk[i], p.sv[i] = a.sv[i], p.sp[i] = a.sp[i], p.so[i] = a.so[i];
  p.tokens = a.tokens;
  p.heads = a.q ? a.heads : 0;
  p.pairs = a.pairs;
  p.naxes = a.naxes;
  p.zero_rest = a.zero_rest;
  return dtype == kF32 ? by_held<float>(cache_dtype, p, a.halves, stream)
                       : dtype == kF16 ? by_held<f16>(cache_dtype, p, a.halves, stream) : by_held<bf16>(cache_dtype, p, a.halves, stream);
}

}  // namespace samhip
