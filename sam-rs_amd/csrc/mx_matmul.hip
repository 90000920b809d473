// Products of microscaled 4-bit matrices on gfx950: out[m, n] = act(sum_k A[m, k] B[n, k] + bias[n]), A and B in blocks of 32
// e2m1 codes under a power of two along k (mx.hpp), sums in f32, out in f32, f16 or bf16, act nothing or the exact GELU.
//
// The matrix units multiply such blocks as they are: v_mfma_scale_f32_32x32x64 takes a lane's 16 bytes (a block of a row)
// and its scale byte. Products of two codes and two scales are exact, so the f32 sums are the only roundings before the
// output's. B is the first operand, so that a lane ends with four consecutive columns of one row of out.
//
// What bounds it: with many rows and a long k, steps whose waves load, read LDS and multiply one after the other, and power: 8192 x
// 8192 of k = 8192 takes 273 us (4.0 PFLOP/s), the units busy in half of the cycles, at 1.8 to 1.9 GHz. The instructions alone, fed
// from registers, would take 127 at 2.4 GHz; with zeros for codes, which take less power, it is 219, so that a third of the gap is
// power. With a short k the results' way out: 4096 x 5120 of k = 1280 in f16 28 us, with
// bias and GELU 35, of which 42 MB of results need 8 and the activation 7. With few rows B's bytes: 7 rows, 1280 columns of
// k = 5120 in f32 6.6 us, a launch, the packing and the way along a row; 16 rows of 8192 to 8192 columns 12.7 (2.8 TB/s of B).
#include <algorithm>

#include "gelu.hpp"
#include "lds_dma.hpp"
#include "mx.hpp"

namespace samhip {

// The rows and columns of the tiles that take least: so many a CU, each its steps and its beginning and end, in ns (what a CU's
// tiles cost together, as one's waits are another's work). Kernel times in f16 by tiles of 64, 128 and 256: 300 x 1280 of k = 5120
// 10.7 and 16.7 us, 4096 x 1280 of 1280 13.4 and 11.4, 4096 x 1280 of 5120 34, 27 and 38, 4096 x 3840 of 1280 30, 22 and 19, 4096 x
// 5120 of 1280 28 and 32 (128, 256), 16001 x 1024 of 4096 49 and 40, 16384 x 4096 of 4096 184 and 156. No tiles of 64, of 256 threads
// each, where a launch would count past 32 bits of them.
int mx_product_tile(int cus, int m, int n, int k) {
  const long steps = (k + 255) / 256;
  auto tiles = [&](long tile) { return (m + tile - 1) / tile * ((n + tile - 1) / tile); };
  auto cost = [&](long tile, long step, long ends) { return (tiles(tile) + cus - 1) / cus * (steps * step + ends); };
  const long large = cost(256, 2100, 5000), middle = cost(128, 670, 2300), small = cost(64, 360, 500);
  if (large < middle && large < small) return 256;
  return middle < small || tiles(64) > (1l << 24) - 8 ? 128 : 64;
}

// Workgroups of the few-row kernel that a CU gets at `blocks` blocks of 16 columns each.
static long few_share(int cus, int n, int blocks) { return ((n + 16l * blocks - 1) / (16l * blocks) + cus - 1) / cus; }
// Two blocks of columns a workgroup, which share what it loads of A, past 8 rows and where no CU gets more columns so: 16 rows of
// 1280 to 5120 columns 3.6 and 3.9 us with two and one, 1 row 3.3 and 3.3; of 8192 to 8192 17 rows 12.2 and 14.5, 32 17.8 and 25.5, 8
// 10.1 and 10.2; of 4096 to 32768 12 rows 18.0 and 19.9, 4 17.3 and 15.9; of 4096 to 11000 (4 and 3 blocks a CU) 16 rows 10.6 and
// 9.3; of 5120 to 1280 6.6 and 5.2.
static int few_blocks(int cus, int m, int n) { return m > 8 && 2 * few_share(cus, n, 2) <= few_share(cus, n, 1) ? 2 : 1; }

// Whether a linear layer's few rows are packed by each workgroup of the few-row kernel again, in place of a launch of their own: up
// to 16 rows while a CU's workgroups pack 8192 values of a row in all, which is also what LDS holds of one. In f16 on the card, so
// and in two launches: 4096 to 4096 columns 1 row 4.5 and 5.8 us, 8 5.7 and 6.4, 16 7.5 and 6.8; 8192 to 4096 8.7 and 8.7 with 8, 11.7
// and 9.8 with 16; 8192 to 8192, where a CU packs once past 8 rows, 12.4 and 12.6 with 9, 14.7 and 14.8 with 16; 4096 to 16384 14.3
// and 12.8 with 16; 5120 to 6144, which takes two up to 8 rows, 7.3 and 8.3 with 4, 9.2 and 8.8 with 8. A launch takes the host 3
// more: called one after the other, 16 rows of 5120 to 8192 take 10.0 and 13.3, of 4096 to 16384 13.9 and 13.3.
bool mx_packs_on_the_way(int m, int n, int k) {
  const int cus = device_cu_count();
  return m <= 16 && few_share(cus, n, few_blocks(cus, m, n)) * k <= 8192;
}

namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ i32x8 codes8(u32x4 w) { return i32x8{(int)w[0], (int)w[1], (int)w[2], (int)w[3], 0, 0, 0, 0}; }

// D(32x32) += A(32x64) B(64x32) of 4-bit codes. Lane l supplies row l % 32 of A and of B^T, block l / 32, and the scales in
// byte SEL of sa and sb; it receives D[8 * (i / 4) + 4 * (l / 32) + i % 4][l % 32] in element i.
template <int SEL> __device__ __forceinline__ f32x16 mma_mx32(u32x4 a, unsigned sa, u32x4 b, unsigned sb, f32x16 c) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(codes8(a), codes8(b), c, 4, 4, SEL, (int)sa, SEL, (int)sb);
}
// D(16x16) += A(16x128) B(128x16): row l % 16, block l / 16, D[4 * (l / 16) + i][l % 16].
__device__ __forceinline__ f32x4 mma_mx16(u32x4 a, unsigned sa, u32x4 b, unsigned sb, f32x4 c) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(codes8(a), codes8(b), c, 4, 4, 0, (int)sa, 0, (int)sb);
}

// Stores columns n .. n + 3 of row m.
template <typename T> __device__ __forceinline__ void put4(const MxProduct& p, int m, int n, f32x4 x, bool whole) {
  if (m >= p.m || n >= p.n) return;
  const T* bias = reinterpret_cast<const T*>(p.bias);
  T* to = reinterpret_cast<T*>(p.out) + (long)m * p.n + n;
  if (whole) {  // n % 4 == 0: whole vectors, aligned
    if (bias) {
      const typename Vec<T>::x4 b = *reinterpret_cast<const typename Vec<T>::x4*>(bias + n);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] += to_f32(b[i]);
    }
    typename Vec<T>::x4 y;
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = from_f32<T>(f32_result(p.gelu ? gelu_for<T>(x[i]) : x[i]));
    *reinterpret_cast<typename Vec<T>::x4*>(to) = y;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (n + i >= p.n) break;
      const float v = x[i] + (bias ? to_f32(bias[n + i]) : 0.f);
      to[i] = from_f32<T>(f32_result(p.gelu ? gelu_for<T>(v) : v));
    }
  }
}

// Many rows. A workgroup of WM x WN waves takes TM x TN of out in steps of 256 along k: rows of 128 bytes, whole cache lines,
// of both matrices go straight to LDS (buffer loads, of which those past a matrix's or row's end bring zeros), the next
// step's while this one is worked on, and come to the matrix units one 16-byte block a lane. 16-byte chunk c of row r lies at
// c ^ (r / 2 % 8), so that the 16 rows of which a read takes a chunk each fall on all 64 banks alike. A row's scales come 16
// bytes at a time, as the loads are bound by the cache lines that they touch: those of two steps where rows of scales are
// whole dwords (k % 128 == 0), else of one step from the dword on in which they begin.
template <typename T, int TM, int TN, int WM, int WN, bool ALIGNED, bool GELU>
__global__ __launch_bounds__(64 * WM * WN) void mx_product_kernel(MxProduct p, int mt, int nt) {
  constexpr int NW = WM * WN, ROWS = TM + TN, CB = ROWS * 128, SB = ROWS * 16;
  constexpr int FM = TM / WM / 32, FN = TN / WN / 32, NC = ROWS / 8 / NW, NG = (ROWS / 64 + NW - 1) / NW;
  static_assert(ROWS % (16 * NW) == 0, "shares of a step");
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
  const unsigned lds0 = lds_addr(smem), lds1 = lds0 + 2 * CB;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // Workgroup i runs on XCD i % 8, whose share of the tiles lies together in bands of GROUP rows of tiles, so that what runs
  // there at once is a block of tiles that share rows of both matrices in its L2
  constexpr int GROUP = 8;
  const int tiles = mt * nt, share = (tiles + 7) / 8, lin = (int)(blockIdx.x % 8) * share + (int)(blockIdx.x / 8);
  if (lin >= tiles) return;
  const int band = lin / (GROUP * nt), rows = min(GROUP, mt - band * GROUP), in = lin - band * GROUP * nt;
  const int m0 = (band * GROUP + in % rows) * TM, n0 = in / rows * TN;
  const int G = p.k / 32, steps = (p.k + 255) / 256;
  const unsigned rb = (unsigned)p.k / 2;  // bytes of a row's codes
  const int mr = min(TM, p.m - m0), nr = min(TN, p.n - n0);
  // rows 0 .. TN - 1 of a step are B's, the others A's
  const i32x4 rsb = buffer_rsrc(p.b + (long)n0 * rb, nr * rb), rsa = buffer_rsrc((const unsigned char*)p.a + (long)m0 * rb, mr * rb);
  // scales in whole dwords: from the one in which the tile's begin to the one in which they end
  const unsigned long sbp = (unsigned long)(p.sb + (long)n0 * G), sap = (unsigned long)(p.sa + (long)m0 * G);
  const unsigned sbo = (unsigned)sbp & 3, sao = (unsigned)sap & 3;
  const i32x4 rssb = buffer_rsrc((const void*)(sbp - sbo), (nr * G + sbo + 3) & ~3u);
  const i32x4 rssa = buffer_rsrc((const void*)(sap - sao), (mr * G + sao + 3) & ~3u);
  auto stage = [&](int t) {
    const unsigned to = lds0 + (t & 1) * CB;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int r0 = 8 * (wave + NW * i);
      const bool of_b = r0 < TN;
      const int chunk = (lane & 7) ^ (lane >> 4) ^ (r0 >> 1 & 4);  // of this lane's row, r0 + lane / 8
      const unsigned off = (unsigned)((of_b ? r0 : r0 - TN) + lane / 8) * rb + 128 * t + 16 * chunk;
      bdma16(of_b ? rsb : rsa, 8 * t + chunk < G ? off : 0x80000000u, to + r0 * 128);  // past the row's end: out of range
    }
    if (ALIGNED && t % 2) return;
#pragma unroll
    for (int i = 0; i < NG; ++i) {
      const int r0 = (64 * (wave + NW * i)) % ROWS;  // waves past the last row bring the first ones again
      const bool of_b = r0 < TN;
      const unsigned off = (unsigned)((of_b ? r0 : r0 - TN) + lane) * (unsigned)G + 8 * t + (of_b ? sbo : sao);
      bdma16(of_b ? rssb : rssa, ALIGNED ? off : off & ~3u, lds1 + ((ALIGNED ? t >> 1 : t) & 1) * SB + r0 * 16);
    }
  };
  const int wm = wave % WM, wn = wave / WM, r = lane & 31, hh = lane >> 5;
  typedef __attribute__((address_space(3))) u32x2 lds_u32x2;
  typedef __attribute__((address_space(3))) u32x4 lds_u32x4;
  const int brow = wn * (TN / WN) + r, arow = TN + wm * (TM / WM) + r;
  const unsigned swz = 16 * (hh ^ (r >> 1 & 7));
  f32x16 acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = f32x16{};
  stage(0);
  for (int t = 0; t < steps; ++t) {
    wait_vm<0>();
    __syncthreads();
    if (t + 1 < steps) stage(t + 1);
    const unsigned at = lds0 + (t & 1) * CB, sat = lds1 + ((ALIGNED ? t >> 1 : t) & 1) * SB;
    // a row's eight scales, those past its end as 2^-127: what came there is another row's, which may be NaN. Then moved so
    // that bytes 0 and 2 of a dword are the lane's.
    const int left = G - 8 * t;
    const unsigned keep[2] = {left >= 4 ? ~0u : (1u << 8 * left) - 1, left >= 8 ? ~0u : left <= 4 ? 0u : (1u << (8 * left - 32)) - 1};
    auto scales_of = [&](int row, unsigned shift) {
      u32x2 s;
      if constexpr (ALIGNED) {
        s = *(const lds_u32x2*)(size_t)(sat + 16 * row + 8 * (t & 1));
      } else {
        const u32x4 w = *(const lds_u32x4*)(size_t)(sat + 16 * row);
        s = u32x2{__builtin_amdgcn_alignbyte(w[1], w[0], shift), __builtin_amdgcn_alignbyte(w[2], w[1], shift)};
      }
      return u32x2{(s[0] & keep[0]) >> (8 * hh), (s[1] & keep[1]) >> (8 * hh)};
    };
    u32x2 sb[FN], sa[FM];
#pragma unroll
    for (int j = 0; j < FN; ++j) sb[j] = scales_of(brow + 32 * j, ((unsigned)(brow + 32 * j) * (unsigned)G + sbo) & 3);
#pragma unroll
    for (int i = 0; i < FM; ++i) sa[i] = scales_of(arow + 32 * i, ((unsigned)(arow - TN + 32 * i) * (unsigned)G + sao) & 3);
#pragma unroll
    for (int q = 0; q < 4; ++q) {  // 64 along k
      u32x4 b[FN], a[FM];
#pragma unroll
      for (int j = 0; j < FN; ++j) b[j] = *(const lds_u32x4*)(size_t)(at + 128 * (brow + 32 * j) + (swz ^ 32 * q));
#pragma unroll
      for (int i = 0; i < FM; ++i) a[i] = *(const lds_u32x4*)(size_t)(at + 128 * (arow + 32 * i) + (swz ^ 32 * q));
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j)
          acc[i][j] = q % 2 ? mma_mx32<2>(b[j], sb[j][q / 2], a[i], sa[i][q / 2], acc[i][j])
                            : mma_mx32<0>(b[j], sb[j][q / 2], a[i], sa[i][q / 2], acc[i][j]);
    }
  }
  __syncthreads();
  // A wave's results go through LDS, 32 rows at a time, so that a row's columns leave together: in f32, 16-byte chunk c of
  // row r at c ^ (r % CH), then V columns a lane with their bias and activation.
  constexpr int COLS = TN / WN, CH = COLS / 4, V = 16 / sizeof(T), LPR = COLS / V, RPP = 64 / LPR;
  const unsigned own = lds0 + wave * (32 * COLS * 4);
  const int n = n0 + wn * COLS + V * (lane % LPR);
  const T* bias = reinterpret_cast<const T*>(p.bias);
  float add[V];
#pragma unroll
  for (int v = 0; v < V; ++v) add[v] = bias && n + v < p.n ? to_f32(bias[n + v]) : 0.f;
  const bool whole = p.n % V == 0;
  typedef __attribute__((address_space(3))) f32x4 lds_f32x4;
#pragma unroll
  for (int i = 0; i < FM; ++i) {
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        *(lds_f32x4*)(size_t)(own + r * (COLS * 4) + 16 * ((8 * j + 2 * e + hh) ^ (r % CH))) =
            f32x4{acc[i][j][4 * e], acc[i][j][4 * e + 1], acc[i][j][4 * e + 2], acc[i][j][4 * e + 3]};
#pragma unroll
    for (int k = 0; k < 32 / RPP; ++k) {
      const int row = RPP * k + lane / LPR, m = m0 + wm * (TM / WM) + 32 * i + row;
      T y[V];
#pragma unroll
      for (int c = 0; c < V / 4; ++c) {
        const f32x4 x = *(const lds_f32x4*)(size_t)(own + row * (COLS * 4) + 16 * ((V / 4 * (lane % LPR) + c) ^ (row % CH)));
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const float z = x[v] + add[4 * c + v];
          y[4 * c + v] = from_f32<T>(f32_result(GELU ? gelu_for<T>(z) : z));
        }
      }
      T* to = reinterpret_cast<T*>(p.out) + (long)m * p.n + n;
      if (m < p.m && n < p.n) {
        if (whole) {
          *reinterpret_cast<u32x4*>(to) = *reinterpret_cast<const u32x4*>(y);
        } else {
#pragma unroll
          for (int v = 0; v < V; ++v)
            if (n + v < p.n) to[v] = y[v];
        }
      }
    }
  }
}

// Few rows: B's bytes bound it, so they go from memory straight to the matrix units. A workgroup takes CB blocks of 16 columns
// of out and RB of 16 rows; its waves take rounds of 512 along k in turn and join at the end, in order. Of a round a lane takes four
// neighbouring blocks of its row, one a step (which blocks meet in a step does not matter while A and B agree): whole lines of a
// row, and four scales in one load (16 rows of k = 5120 to 1280 columns 5.2 us, 6.7 with neighbouring blocks in neighbouring
// lanes; 16384 to 1024 11.3 and 16.5; 8192 to 8192 12.7 and 17.0; 8 or 4 columns a workgroup, for more of them, change nothing).
// RAW: A comes as it is, and each workgroup packs it into LDS first.
template <typename T, int RB, int CB, bool RAW>
__global__ __launch_bounds__(1024) void mx_few_kernel(MxProduct p) {
  constexpr int U = 4;  // steps in flight, and bytes of a load of scales
  __shared__ __attribute__((aligned(16))) f32x4 part[16][CB * RB][64];
  extern __shared__ __attribute__((aligned(16))) unsigned char packed[];  // [m][k / 2] codes, then [m][k / 32] scales
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const int r = lane & 15, g = lane >> 4, n0 = 16 * CB * blockIdx.x;
  const int G = p.k / 32;
  const long rb = p.k / 2;
  const unsigned char *br[CB], *bs[CB];
#pragma unroll
  for (int j = 0; j < CB; ++j) {
    const int column = min(n0 + 16 * j + r, p.n - 1);
    br[j] = p.b + column * rb;
    bs[j] = p.sb + column * (long)G;
  }
  const unsigned char* a0 = RAW ? packed : reinterpret_cast<const unsigned char*>(p.a);
  const unsigned char* sa0 = RAW ? packed + p.m * (p.k / 2) : p.sa;
  const unsigned char *ar[RB], *as[RB];
#pragma unroll
  for (int i = 0; i < RB; ++i) {
    ar[i] = a0 + min(16 * i + r, p.m - 1) * rb;
    as[i] = sa0 + min(16 * i + r, p.m - 1) * (long)G;
  }
  if constexpr (RAW) {
    const int vectors = p.m * (p.k / 8), rounds = (vectors + blockDim.x - 1) / blockDim.x;  // of 8 values, a quad a block
    for (int v0 = 0; v0 < rounds; v0 += U) {
      Eight<T> x[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        x[u] = load_eight(reinterpret_cast<const T*>(p.a) + 8l * min((int)threadIdx.x + (v0 + u) * (int)blockDim.x, vectors - 1));
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int at = threadIdx.x + (v0 + u) * blockDim.x;
        unsigned s;
        const unsigned w = mx_quantise(x[u], s);
        if (at < vectors) {
          reinterpret_cast<unsigned*>(packed)[at] = w;
          if (at % 4 == 0) packed[p.m * (p.k / 2) + at / 4] = (unsigned char)s;
        }
      }
    }
    __syncthreads();
  }
  f32x4 acc[CB][RB];
#pragma unroll
  for (int j = 0; j < CB; ++j)
#pragma unroll
    for (int i = 0; i < RB; ++i) acc[j][i] = f32x4{};
  // a lane's U blocks of a round follow one another, so that their scales are one load where no row ends inside it
  auto scales_of = [&](const unsigned char* p, int c) {
    unsigned s = 0;
    if (G % U == 0) {
      __builtin_memcpy(&s, p + min(c, G - U), U);  // scales may begin at any byte
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u) s |= (unsigned)p[min(c + u, G - 1)] << (8 * u);
    }
    return s;
  };
  for (int c0 = 4 * U * wave; c0 < G; c0 += 4 * U * waves) {
    const int c = c0 + U * g;
    u32x4 b[U][CB], a[U][RB];
    unsigned sb[CB], sa[RB];
#pragma unroll
    for (int j = 0; j < CB; ++j) sb[j] = scales_of(bs[j], c);
#pragma unroll
    for (int i = 0; i < RB; ++i) sa[i] = scales_of(as[i], c);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int at = 16 * min(c + u, G - 1);
#pragma unroll
      for (int j = 0; j < CB; ++j) b[u][j] = *reinterpret_cast<const u32x4*>(br[j] + at);
#pragma unroll
      for (int i = 0; i < RB; ++i) a[u][i] = *reinterpret_cast<const u32x4*>(ar[i] + at);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool in = c + u < G;  // blocks past the row's end: zeros under 2^-127
#pragma unroll
      for (int j = 0; j < CB; ++j) {
        const u32x4 bu = in ? b[u][j] : u32x4{};
#pragma unroll
        for (int i = 0; i < RB; ++i)
          acc[j][i] = mma_mx16(bu, in ? sb[j] >> (8 * u) & 255 : 0u, a[u][i], in ? sa[i] >> (8 * u) & 255 : 0u, acc[j][i]);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < CB; ++j)
#pragma unroll
    for (int i = 0; i < RB; ++i) part[wave][j * RB + i][lane] = acc[j][i];
  __syncthreads();
  for (int i = wave; i < CB * RB; i += waves) {
    f32x4 x = part[0][i][lane];
    for (int w = 1; w < waves; ++w) x += part[w][i][lane];
    put4<T>(p, 16 * (i % RB) + r, n0 + 16 * (i / RB) + 4 * g, x, p.n % 4 == 0);
  }
}

template <typename T, int TM, int TN, int WM, int WN, bool ALIGNED, bool GELU>
hipError_t launch_product(const MxProduct& p, hipStream_t stream) {
  constexpr int lds = 2 * (TM + TN) * (128 + 16);
  static_assert(lds >= WM * WN * 32 * (TN / WN) * 4, "the results' way out");
  auto kern = mx_product_kernel<T, TM, TN, WM, WN, ALIGNED, GELU>;
  static std::atomic<unsigned long long> done;
  if (const hipError_t e = lds_opt_in(done, (const void*)kern, lds); e != hipSuccess) return e;
  const int mt = (p.m + TM - 1) / TM, nt = (p.n + TN - 1) / TN;
  const long grid = ((long)mt * nt + 7) / 8 * 8;
  hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(64 * WM * WN), lds, stream, p, mt, nt);
  return hipGetLastError();
}
template <typename T, int TM, int TN, int WM, int WN> hipError_t by_alignment(const MxProduct& p, hipStream_t stream) {
  if (p.k % 128 == 0 && reinterpret_cast<uintptr_t>(p.sa) % 4 == 0 && reinterpret_cast<uintptr_t>(p.sb) % 4 == 0)
    return p.gelu ? launch_product<T, TM, TN, WM, WN, true, true>(p, stream) : launch_product<T, TM, TN, WM, WN, true, false>(p, stream);
  return p.gelu ? launch_product<T, TM, TN, WM, WN, false, true>(p, stream) : launch_product<T, TM, TN, WM, WN, false, false>(p, stream);
}

constexpr int kMostPacked = 16 * (8192 / 2 + 8192 / 32);  // bytes of LDS

template <typename T, int CB> hipError_t few(const MxProduct& p, hipStream_t stream) {
  // a wave for each round: 16 rows of k = 5120 to 1280 columns 5.2 us with 10, 6.7, 5.5, 5.4, 5.3 and 5.4 with 1, 2, 4, 8 and 16; of
  // 1280 to 5120 3.8 with 3, 4.1, 3.9, 3.9, 4.1 and 4.2
  const int waves = (int)std::min(16, std::max(1, (p.k + 511) / 512));
  const dim3 grid((unsigned)((p.n + 16 * CB - 1) / (16 * CB)));
  if (!p.sa) {
    const int lds = p.m * (p.k / 2 + p.k / 32);
    static std::atomic<unsigned long long> done;
    if (const hipError_t e = lds_opt_in(done, (const void*)mx_few_kernel<T, 1, CB, true>, kMostPacked); e != hipSuccess) return e;
    hipLaunchKernelGGL((mx_few_kernel<T, 1, CB, true>), grid, dim3(64 * waves), lds, stream, p);
  } else if (p.m <= 16)
    hipLaunchKernelGGL((mx_few_kernel<T, 1, CB, false>), grid, dim3(64 * waves), 0, stream, p);
  else
    hipLaunchKernelGGL((mx_few_kernel<T, 2, CB, false>), grid, dim3(64 * waves), 0, stream, p);
  return hipGetLastError();
}

template <typename T> hipError_t product(const MxProduct& p, hipStream_t stream) {
  const int cus = device_cu_count();
  if (p.m <= 32) return few_blocks(cus, p.m, p.n) == 2 ? few<T, 2>(p, stream) : few<T, 1>(p, stream);
  const int tile = mx_product_tile(cus, p.m, p.n, p.k);
  if (tile == 256) return by_alignment<T, 256, 256, 2, 4>(p, stream);
  return tile == 128 ? by_alignment<T, 128, 128, 2, 2>(p, stream) : by_alignment<T, 64, 64, 2, 2>(p, stream);
}

}  // namespace

hipError_t mx_matmul(int dtype, const MxProduct& p, hipStream_t stream) {
  if (p.m == 0 || p.n == 0) return hipSuccess;
  return dtype == kF32 ? product<float>(p, stream) : dtype == kF16 ? product<f16>(p, stream) : product<bf16>(p, stream);
}

}  // namespace samhip
