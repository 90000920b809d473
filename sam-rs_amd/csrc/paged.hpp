// Host/device interface of the paged key/value memory: the cache's pages (kv_cache.hip) and the attention of new
// tokens over them (paged_attn*.hip).
//
// A pool holds pages [pages, heads, page_size, d] of keys and another of values. Sequence b's key j lies in page
// table[b][j / page_size], slot j % page_size. In 8 bits (e4m3) a row of d values has one scale, a power of two held
// as its biased exponent: value = code * 2^(scale - 127).
#pragma once
#include "common.hpp"

namespace samhip {

constexpr int kE4M3 = 3;  // cache dtype code beside DType's
struct e4m3 {
  unsigned char bits;
};

struct PagedKv {
  void* k;
  void* v;
  unsigned char* ks;  // scales [pages, heads, page_size], e4m3 only
  unsigned char* vs;
  const int* table;   // [batch, width]
  const int* starts;  // [batch + 1] first token of each sequence among the new ones (null: kv_read)
  const int* lens;    // [batch] tokens that each sequence holds, the new ones included
  int batch, pages, heads, page, d, width;
  unsigned magic, shift;  // j / page == (j * magic) >> shift for 0 <= j < 2^31
};

// j / d by a multiplication: with L = ceil(log2 d) and m = floor(2^(31 + L) / d) + 1, m exceeds 2^(31+L) / d by at
// most 1 <= 2^L / d, i.e. by 2^-31 of itself at most, which is exact for every j below 2^31.
inline void division_magic(int d, unsigned* magic, unsigned* shift) {
  unsigned l = 0;
  while ((1l << l) < d) ++l;
  *shift = 31 + l;
  *magic = (unsigned)((1ul << (31 + l)) / (unsigned)d + 1);
}
__host__ __device__ inline unsigned divide_magic(unsigned j, unsigned magic, unsigned shift) {
  return (unsigned)(((unsigned long)j * magic) >> shift);
}

// Where sequence b's key j lies for one head: first the table's entry, a load that is best on its way long before it is
// needed, then the row (of the pools seen as [pages * heads * page_size, d], fewer than 2^31 of them), -1 where j is past
// `end` or the entry outside the pool.
struct PagedEntry {
  int page, slot;
};
__device__ __forceinline__ PagedEntry paged_entry(const PagedKv& c, int b, int j, int end) {
  const int at = max(0, min(j, end - 1));
  const unsigned t = divide_magic((unsigned)at, c.magic, c.shift);
  return {c.table[(long)b * c.width + t], at == j ? at - (int)t * c.page : -1};
}
__device__ __forceinline__ int paged_row(const PagedKv& c, const PagedEntry& e, int head) {
  return (unsigned)e.page < (unsigned)c.pages && e.slot >= 0 ? (e.page * c.heads + head) * c.page + e.slot : -1;
}
__device__ __forceinline__ int paged_row(const PagedKv& c, int b, int head, int j, int end) {
  return (unsigned)j < (unsigned)end ? paged_row(c, paged_entry(c, b, j, end), head) : -1;
}

// Keys that sequence b holds, inside what its table can name.
__device__ __forceinline__ int paged_len(const PagedKv& c, int b) {
  return max(0, min(c.lens[b], c.width * c.page));
}

__device__ __forceinline__ float pow2_of(unsigned char biased) {
  return __uint_as_float(biased ? (unsigned)biased << 23 : 0x00400000u);  // 2^-127 is subnormal
}

// Arguments of one paged-attention launch. Strides in elements: [0] token, [1] head.
struct PagedParams {
  PagedKv c;
  const void* q;
  void* out;
  long sq[2], so[2];
  int tokens, heads, group;   // query heads, and how many of them share a key head
  unsigned gmagic, gshift;    // division by group
  float sc;                   // scale * log2(e)
  int causal, zero_rest;
  int rtiles, nsplit;         // row tiles per (sequence, key head) of the grid; key splits
  int round;                  // row tiles of one workgroup a CU (0: less than one)
  int per;                    // blocks of 32 keys per split, at least (0: even shares of what each sequence holds)
  float* opart;               // nsplit > 1: partial O [nsplit][tokens * heads][d], f32, not normalised
  float* ml;                  // nsplit > 1: running (max, sum) [nsplit][tokens * heads][2], log2 units; a sum of -1 in
                              // split 0: the row is finished, the other splits have written nothing
};

// How a call runs: the kernel's rows per tile, the row tiles and key splits of its grid, its workspace.
struct PagedPlan {
  int many, rows, rtiles, nsplit, per, round;
  long part_bytes, total;
};
PagedPlan paged_plan(int dtype, int cache_dtype, int tokens, int batch, int heads, int kv_heads, int d, int max_q,
                     int max_len, int cus);
hipError_t paged_attention(int dtype, int cache_dtype, PagedParams p, const PagedPlan& plan, hipStream_t stream);
hipError_t paged_f32(int cache_dtype, const PagedParams& p, int rows, hipStream_t stream);
hipError_t paged_few(int dtype, int cache_dtype, const PagedParams& p, int rows, hipStream_t stream);
hipError_t paged_many(int dtype, int cache_dtype, const PagedParams& p, hipStream_t stream);
hipError_t paged_combine(int dtype, const PagedParams& p, hipStream_t stream);

hipError_t kv_write(int dtype, int cache_dtype, const void* k, const void* v, const long* sk, const long* sv,
                    const PagedKv& c, int tokens, hipStream_t stream);
hipError_t kv_read(int dtype, int cache_dtype, void* k, void* v, const PagedKv& c, int max_len, hipStream_t stream);

hipError_t rope_axes(int dtype, const void* x, const int* pos, const double* freqs, const int* axes, void* out, int b,
                     int l, int h, int d, int pairs, int naxes, const long* sx, const long* sp, const long* so,
                     int halves, int inverse, hipStream_t stream);

// ------------------------------------------------------------------------------------------ device helpers

// Two codes (the low or the high half of w) times a power of two, as a pair of T.
template <typename T, bool HI> __device__ __forceinline__ unsigned decode2(unsigned w, float s);
template <> __device__ __forceinline__ unsigned decode2<f16, false>(unsigned w, float s) {
  return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, s, false));
}
template <> __device__ __forceinline__ unsigned decode2<f16, true>(unsigned w, float s) {
  return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, s, true));
}
template <> __device__ __forceinline__ unsigned decode2<bf16, false>(unsigned w, float s) {
  return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w, s, false));
}
template <> __device__ __forceinline__ unsigned decode2<bf16, true>(unsigned w, float s) {
  return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w, s, true));
}

// Bits 15 and 31 of the result say which 16-bit halves of w are infinite or NaN: their exponent bits, all ones, carry.
template <typename T> __device__ __forceinline__ unsigned not_finite2(unsigned w) {
  constexpr unsigned e = __is_same(T, f16) ? 0x7c00u : 0x7f80u, one = __is_same(T, f16) ? 0x0400u : 0x0080u;
  return ((w & (e | e << 16)) + (one | one << 16)) & 0x80008000u;
}
// w without those halves.
__device__ __forceinline__ unsigned without2(unsigned w, unsigned bad) {
  return w & ~((bad >> 15) * 0xffffu);
}

// Four values of a cache row in T (each rounded to it), as f32: those that are not finite, and 0 for the others.
template <typename T, typename C> __device__ __forceinline__ f32x4 only_not_finite4(const C* p, float s) {
  u32x2 x;
  if constexpr (__is_same(C, e4m3)) {
    const unsigned w = *reinterpret_cast<const unsigned*>(p);
    x = u32x2{decode2<T, false>(w, s), decode2<T, true>(w, s)};
  } else {
    x = *reinterpret_cast<const u32x2*>(p);
  }
  const typename Vec<T>::x4 v = __builtin_bit_cast(typename Vec<T>::x4, x);
  f32x4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float f = to_f32(v[i]);
    r[i] = fabsf(f) < INFINITY ? 0.f : f;
  }
  return r;
}

// One sequence's new tokens [s0, s0 + lq), keys, and the row tile this workgroup starts with. Its token t sits at position
// before + t, where kv_write puts it: behind the table's end too, if lens passes that.
struct PagedWork {
  int tile, split, head, b;
  int s0, lq, len, before;
};
// Keys that token t of a sequence sees, of those it holds.
__device__ __forceinline__ int paged_keys(const PagedWork& w, int causal, int t) {
  return causal ? max(0, min(w.len, w.before + t + 1)) : w.len;
}
__device__ __forceinline__ PagedWork paged_work(const PagedParams& p) {
  // Workgroup i runs on XCD i % 8. The (sequence, key head) comes first, then the key split, the row tile last: a
  // multiple of 8 of the first two leaves each head's keys to one XCD's L2, and sequences of different lengths, whose
  // heads are neighbours, spread over all XCDs.
  const int units = p.c.heads * p.c.batch, lin = blockIdx.x, unit = lin % units;
  PagedWork w;
  w.split = lin / units % p.nsplit;
  w.tile = lin / (units * p.nsplit);
  if (p.causal) {
    // The tiles with most keys first, and every second round of one workgroup a CU in the other order, so that a CU's
    // first two have as many keys together as any other's (workgroups i and i + 256 share a CU; 8192 tokens over their own
    // keys, 8 heads of 128 in f16: 252 -> 227 us; 4 sequences of 2048 in bf16: 88 -> 81).
    if (p.round > 0) {
      const int from = w.tile / p.round * p.round, many = min(p.round, p.rtiles - from);
      if (w.tile / p.round & 1) w.tile = 2 * from + many - 1 - w.tile;
    }
    w.tile = p.rtiles - 1 - w.tile;
  }
  w.head = unit % p.c.heads;
  w.b = unit / p.c.heads;
  const int end = p.c.starts[w.b + 1], held = p.c.lens[w.b];
  w.s0 = max(0, min(p.c.starts[w.b], p.tokens));
  w.lq = max(0, min(end, p.tokens) - w.s0);
  w.len = paged_len(p.c, w.b);
  // 64 bits, for any lens and starts: before + lq <= lens, and what is below -2^31 sees no key either way
  w.before = (int)max((long)held - end + w.s0, -(1l << 31));
  return w;
}

// Key blocks of a split where n are shared out in pieces of `most` at best, `splits` pieces at most: even ones.
__device__ __forceinline__ int paged_share(int n, int most, int splits) {
  const int per = max(max(most, 1), (n + splits - 1) / splits), pieces = max(1, (n + per - 1) / per);
  return (n + pieces - 1) / pieces;
}

// Sets the rows of out that belong to no sequence to zero, spread over the launch's workgroups.
template <typename T> __device__ __forceinline__ void paged_zero_rest(const PagedParams& p) {
  const int first = max(0, min(p.c.starts[0], p.tokens)), end = max(first, min(p.c.starts[p.c.batch], p.tokens));
  const int rest = p.tokens - (end - first), cols = p.heads * (p.c.d / 8);
  for (int i = blockIdx.x; i < rest; i += gridDim.x) {
    const long t = i < first ? i : end + (i - first);
    for (int c = threadIdx.x; c < cols; c += blockDim.x) {
      const int head = c / (p.c.d / 8), col = c % (p.c.d / 8) * 8;
      u32x4* w = reinterpret_cast<u32x4*>(reinterpret_cast<T*>(p.out) + t * p.so[0] + head * p.so[1] + col);
      w[0] = u32x4{};
      if (sizeof(T) == 4) w[1] = u32x4{};
    }
  }
}

}  // namespace samhip
