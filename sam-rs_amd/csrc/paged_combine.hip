// Joins the key splits of a paged-attention call on gfx950: out = sum_s O_s 2^(m_s - M) / sum_s l_s 2^(m_s - M), M the
// largest m_s of the row, from the partial results that the attention kernels left. Splits are added in order, so the
// result does not depend on their timing. A split without keys has l = 0 and no O; a row whose keys are all in its
// first split is written already, which l = -1 says.
//
// What bounds it: the partial O's bytes, 4 a column and split, and, with few rows, the latency of reading them. A thread
// reads its four columns of each split, eight of them at a time; past eight splits and while there are few rows a
// workgroup takes 32 columns of a row, its lanes a share of the splits each, and they meet in LDS (16 rows of 128 columns
// and 256 splits: 15.4 us with a lane for each 4 columns and a wave for each 32 splits, 4.1 so).
#include "paged.hpp"

namespace samhip {

namespace {

__device__ __forceinline__ bool row_of_a_sequence(const PagedParams& p, int tok) {
  return tok >= p.c.starts[0] && tok < p.c.starts[p.c.batch];  // the others have no partial results
}

template <typename T> __device__ __forceinline__ void store_row4(const PagedParams& p, int tok, int head, int col,
                                                                 f32x4 o, float l) {
  const float inv = l == 0.f ? 0.f : 1.f / l;  // a row that sees no key is 0
  typename Vec<T>::x4 x;
#pragma unroll
  for (int j = 0; j < 4; ++j) x[j] = from_f32<T>(f32_result(o[j] * inv));
  *reinterpret_cast<typename Vec<T>::x4*>(reinterpret_cast<T*>(p.out) + tok * p.so[0] + head * p.so[1] + col) = x;
}

// A thread takes 4 columns of a row and up to N splits: all their maxima and sums are on their way together, then all
// their partial results (4096 rows of 256 and 8 splits: 11.0 us one after the other, 7.9 so).
template <typename T, int N> __global__ __launch_bounds__(256) void paged_combine_kernel(PagedParams p) {
  const unsigned cpr = p.c.d / 4, i = blockIdx.x * 256u + threadIdx.x;  // fewer than 2^32 threads
  const unsigned row = i / cpr;
  const int col = (int)(i - row * cpr) * 4;
  const long rows = (long)p.tokens * p.heads;
  if (row >= rows) return;
  const int tok = (int)(row / (unsigned)p.heads), head = (int)(row - tok * (unsigned)p.heads);
  float2 ml[N];
#pragma unroll
  for (int s = 0; s < N; ++s) ml[s] = *reinterpret_cast<const float2*>(p.ml + 2 * (min(s, p.nsplit - 1) * rows + row));
  if (!row_of_a_sequence(p, tok) || ml[0].y < 0.f) return;
  f32x4 x[N];
#pragma unroll
  for (int s = 0; s < N; ++s) {
    x[s] = *reinterpret_cast<const f32x4*>(p.opart + (min(s, p.nsplit - 1) * rows + row) * p.c.d + col);
    if (s >= p.nsplit) ml[s] = float2{-INFINITY, 0.f};
  }
  float top = ml[0].x;
#pragma unroll
  for (int s = 1; s < N; ++s) top = fmaxf(top, ml[s].x);
  const float base = top == -INFINITY ? 0.f : top;
  f32x4 o = {};
  float l = 0.f;
#pragma unroll
  for (int s = 0; s < N; ++s) {
    const float w = exp2_fast(ml[s].x - base);
    l += ml[s].y == 0.f ? 0.f : ml[s].y * w;
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] += ml[s].y == 0.f ? 0.f : x[s][j] * w;  // no keys in this split: its O was not written
  }
  store_row4<T>(p, tok, head, col, o, l);
}

// The same for more splits, eight of them at a time.
template <typename T> __global__ __launch_bounds__(256) void paged_combine_long_kernel(PagedParams p) {
  const unsigned cpr = p.c.d / 4, i = blockIdx.x * 256u + threadIdx.x;  // fewer than 2^32 threads
  const unsigned row = i / cpr;
  const int col = (int)(i - row * cpr) * 4;
  const long rows = (long)p.tokens * p.heads;
  if (row >= rows) return;
  const int tok = (int)(row / (unsigned)p.heads), head = (int)(row - tok * (unsigned)p.heads);
  float2 ml[8];
  auto load_ml = [&](int s0) {
#pragma unroll
    for (int k = 0; k < 8; ++k) ml[k] = *reinterpret_cast<const float2*>(p.ml + 2 * (min(s0 + k, p.nsplit - 1) * rows + row));
  };
  load_ml(0);
  if (!row_of_a_sequence(p, tok) || ml[0].y < 0.f) return;
  float top = -INFINITY;
  for (int s0 = 0; s0 < p.nsplit; s0 += 8) {
    load_ml(s0);
#pragma unroll
    for (int k = 0; k < 8; ++k) top = fmaxf(top, ml[k].x);
  }
  const float base = top == -INFINITY ? 0.f : top;
  f32x4 o = {};
  float l = 0.f;
  for (int s0 = 0; s0 < p.nsplit; s0 += 8) {
    load_ml(s0);
    f32x4 x[8];
#pragma unroll
    for (int k = 0; k < 8; ++k)
      x[k] = *reinterpret_cast<const f32x4*>(p.opart + (min(s0 + k, p.nsplit - 1) * rows + row) * p.c.d + col);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const bool none = s0 + k >= p.nsplit || ml[k].y == 0.f;  // no keys in this split: its O was not written
      const float w = exp2_fast(ml[k].x - base);
      l += none ? 0.f : ml[k].y * w;
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] += none ? 0.f : x[k][j] * w;
    }
  }
  store_row4<T>(p, tok, head, col, o, l);
}

constexpr int kRowWaves = 8, kMostSplits = 256, kCols = 32;

// A workgroup takes 32 columns of a row: 8 lanes' 16 bytes of 64 splits at a time. Every partial result is on its way
// before the weights are known, so that the two dependent reads overlap.
template <typename T> __global__ __launch_bounds__(64 * kRowWaves) void paged_combine_row_kernel(PagedParams p) {
  constexpr int kDeep = kMostSplits / (8 * kRowWaves);
  __shared__ float weight[kMostSplits], red[2][kRowWaves];
  __shared__ __attribute__((aligned(16))) f32x4 part[kRowWaves][8];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int groups = (p.c.d + kCols - 1) / kCols;
  const unsigned row = blockIdx.x / (unsigned)groups;
  const long rows = (long)p.tokens * p.heads;
  const int tok = (int)(row / (unsigned)p.heads), head = (int)(row - tok * (unsigned)p.heads);
  if (!row_of_a_sequence(p, tok) || p.ml[2l * row + 1] < 0.f) return;
  const int col = (int)(blockIdx.x % groups) * kCols + 4 * (lane & 7), s0 = 8 * wave + (lane >> 3);
  f32x4 x[kDeep];
#pragma unroll
  for (int k = 0; k < kDeep; ++k) {
    const long s = min(s0 + 64 * k, p.nsplit - 1);
    if (64 * k < p.nsplit) x[k] = *reinterpret_cast<const f32x4*>(p.opart + (s * rows + row) * p.c.d + min(col, p.c.d - 4));
  }
  const int s = threadIdx.x;
  float2 ml = {-INFINITY, 0.f};
  if (s < p.nsplit) ml = *reinterpret_cast<const float2*>(p.ml + 2 * (s * rows + row));
  float top = ml.x;
#pragma unroll
  for (int k = 1; k < 64; k *= 2) top = fmaxf(top, __shfl_xor(top, k));
  if (lane == 0) red[0][wave] = top;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kRowWaves; ++k) top = fmaxf(top, red[0][k]);
  const float base = top == -INFINITY ? 0.f : top;
  const float w = ml.y == 0.f ? 0.f : exp2_fast(ml.x - base);
  if (s < kMostSplits) weight[s] = ml.y == 0.f ? -1.f : w;  // -1: no keys, its O was not written
  float l = ml.y == 0.f ? 0.f : ml.y * w;
#pragma unroll
  for (int k = 1; k < 64; k *= 2) l += __shfl_xor(l, k);
  if (lane == 0) red[1][wave] = l;
  __syncthreads();
  l = 0.f;
#pragma unroll
  for (int k = 0; k < kRowWaves; ++k) l += red[1][k];
  f32x4 o = {};
#pragma unroll
  for (int k = 0; k < kDeep; ++k) {
    if (64 * k < p.nsplit) {
      const float f = weight[s0 + 64 * k];
      if (f != -1.f) o += x[k] * f;
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int k = 8; k < 64; k *= 2) o[j] += __shfl_xor(o[j], k);
  if (lane < 8) part[wave][lane] = o;
  __syncthreads();
  if (threadIdx.x >= 8 || col >= p.c.d) return;
#pragma unroll
  for (int k = 1; k < kRowWaves; ++k) o += part[k][lane];
  store_row4<T>(p, tok, head, col, o, l);
}

// A workgroup for 32 columns of a row while there are few rows: with 12 splits, attention of 4000 rows of 128 and joining
// take 73 us so and 31 with threads, of 800 rows of 64 17.5 and 14.1, of 400 of 128 (32 splits) 29.9 and 29.7.
constexpr long kMostBlocks = 1024;

template <typename T> hipError_t combine(const PagedParams& p, hipStream_t stream) {
  const long rows = (long)p.tokens * p.heads;
  const long blocks = rows * ((p.c.d + kCols - 1) / kCols);
  const long threads = rows * (p.c.d / 4);
  if (p.nsplit > 8 && blocks > kMostBlocks) {
    hipLaunchKernelGGL(paged_combine_long_kernel<T>, dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, stream, p);
  } else if (p.nsplit > 8) {
    static_assert(kMostSplits <= 64 * kRowWaves, "a thread for each split");
    hipLaunchKernelGGL(paged_combine_row_kernel<T>, dim3((unsigned)blocks), dim3(64 * kRowWaves), 0, stream, p);
  } else {
    auto kern = p.nsplit <= 2 ? paged_combine_kernel<T, 2> : p.nsplit <= 4 ? paged_combine_kernel<T, 4> : paged_combine_kernel<T, 8>;
    hipLaunchKernelGGL(kern, dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, stream, p);
  }
  return hipGetLastError();
}

}  // namespace

hipError_t paged_combine(int dtype, const PagedParams& p, hipStream_t stream) {
  return dtype == kF32 ? combine<float>(p, stream) : dtype == kF16 ? combine<f16>(p, stream) : combine<bf16>(p, stream);
}

}  // namespace samhip
