// Rows into microscaled 4-bit numbers and back, on gfx950 (mx.hpp has the format).
//
// What bounds both: HBM bytes, a value in and its 4 bits out. A lane takes 8 values (16-byte loads of 16-bit ones), so that
// the four lanes of a quad have a block and find its largest magnitude in two exchanges inside the quad; the scale is a
// shift of that one's exponent, and one conversion instruction a pair of values divides and rounds.
#include "mx.hpp"

namespace samhip {

namespace {

// A thread takes U vectors of 8 values, a workgroup's threads a run of 256 neighbours each time.
template <typename T, int U>
__global__ __launch_bounds__(256) void mx_pack_kernel(const T* x, unsigned* codes, unsigned char* scales, long vectors) {
  const long first = (long)blockIdx.x * (256 * U) + threadIdx.x;
  Eight<T> v[U];
#pragma unroll
  for (int u = 0; u < U; ++u) v[u] = load_eight(x + 8 * min(first + 256 * u, vectors - 1));
#pragma unroll
  for (int u = 0; u < U; ++u) {
    unsigned s;
    const unsigned w = mx_quantise(v[u], s);
    const long at = first + 256 * u;
    if (at < vectors) {
      codes[at] = w;
      if ((threadIdx.x & 3) == 0) scales[at >> 2] = (unsigned char)s;
    }
  }
}

template <typename T, int U>
__global__ __launch_bounds__(256) void mx_unpack_kernel(const unsigned* codes, const unsigned char* scales, T* x, long vectors) {
  const long first = (long)blockIdx.x * (256 * U) + threadIdx.x;
  unsigned w[U];
  unsigned char s[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const long at = min(first + 256 * u, vectors - 1);
    w[u] = codes[at];
    s[u] = scales[at >> 2];
  }
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (first + 256 * u < vectors) store_eight(x + 8 * (first + 256 * u), mx_dequantise<T>(w[u], mx_scale(s[u])));
}

template <typename T> hipError_t pack(const void* x, unsigned char* codes, unsigned char* scales, long vectors, hipStream_t stream) {
  const T* from = reinterpret_cast<const T*>(x);
  unsigned* to = reinterpret_cast<unsigned*>(codes);
  if (vectors >= 1l << 18)
    hipLaunchKernelGGL((mx_pack_kernel<T, 4>), dim3((unsigned)((vectors + 1023) / 1024)), dim3(256), 0, stream, from, to, scales, vectors);
  else
    hipLaunchKernelGGL((mx_pack_kernel<T, 1>), dim3((unsigned)((vectors + 255) / 256)), dim3(256), 0, stream, from, to, scales, vectors);
  return hipGetLastError();
}
template <typename T> hipError_t unpack(const unsigned char* codes, const unsigned char* scales, void* x, long vectors, hipStream_t stream) {
  const unsigned* from = reinterpret_cast<const unsigned*>(codes);
  T* to = reinterpret_cast<T*>(x);
  if (vectors >= 1l << 18)
    hipLaunchKernelGGL((mx_unpack_kernel<T, 4>), dim3((unsigned)((vectors + 1023) / 1024)), dim3(256), 0, stream, from, scales, to, vectors);
  else
    hipLaunchKernelGGL((mx_unpack_kernel<T, 1>), dim3((unsigned)((vectors + 255) / 256)), dim3(256), 0, stream, from, scales, to, vectors);
  return hipGetLastError();
}

}  // namespace

hipError_t mx_pack(int dtype, const void* x, unsigned char* codes, unsigned char* scales, long blocks, hipStream_t stream) {
  if (blocks == 0) return hipSuccess;
  return dtype == kF32 ? pack<float>(x, codes, scales, 4 * blocks, stream)
                       : dtype == kF16 ? pack<f16>(x, codes, scales, 4 * blocks, stream) : pack<bf16>(x, codes, scales, 4 * blocks, stream);
}
hipError_t mx_unpack(int dtype, const unsigned char* codes, const unsigned char* scales, void* x, long blocks, hipStream_t stream) {
  if (blocks == 0) return hipSuccess;
  return dtype == kF32 ? unpack<float>(codes, scales, x, 4 * blocks, stream)
                       : dtype == kF16 ? unpack<f16>(codes, scales, x, 4 * blocks, stream) : unpack<bf16>(codes, scales, x, 4 * blocks, stream);
}

}  // namespace samhip
