// Rows into microscaled 4-bit numbers and back, on gfx950 (mx.hpp has the format).
//
// What bounds both: HBM bytes, a value in and its 4 bits out. A lane takes 8 values (16-byte loads of 16-bit ones), so that
// the four lanes of a quad have a block and find its largest magnitude in two exchanges inside the quad; the scale is a
// shift of that one's exponent, and one conversion instruction a pair of values divides and rounds.
//
// Measured, 16384 rows of 8192 in bf16: packed in 57 us (5.9 TB/s), unpacked in 58 (5.8); a copy of 1 GiB reaches 5.2. 196
// rows of 1280 in f32 are a launch, 2.3 us.
#include "mx.hpp"

namespace samhip {

namespace {

template <typename T>
__global__ __launch_bounds__(256) void mx_pack_kernel(const T* x, unsigned* codes, unsigned char* scales, long vectors) {
  const long at = (long)blockIdx.x * 256 + threadIdx.x;
  unsigned s;
  const unsigned w = mx_quantise(load_eight(x + 8 * min(at, vectors - 1)), s);
  if (at >= vectors) return;
  codes[at] = w;
  if ((threadIdx.x & 3) == 0) scales[at >> 2] = (unsigned char)s;
}

// A thread takes U vectors of 8 values, a workgroup's threads a run of 256 neighbours each time.
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
  hipLaunchKernelGGL(mx_pack_kernel<T>, dim3((unsigned)((vectors + 255) / 256)), dim3(256), 0, stream, reinterpret_cast<const T*>(x),
                     reinterpret_cast<unsigned*>(codes), scales, vectors);
  return hipGetLastError();
}
template <typename T, int U>
hipError_t launch_unpack(const unsigned char* codes, const unsigned char* scales, void* x, long vectors, hipStream_t stream) {
  hipLaunchKernelGGL((mx_unpack_kernel<T, U>), dim3((unsigned)((vectors + 256 * U - 1) / (256 * U))), dim3(256), 0, stream,
                     reinterpret_cast<const unsigned*>(codes), scales, reinterpret_cast<T*>(x), vectors);
  return hipGetLastError();
}
// Four vectors a thread for 16-bit values of 256 MB on, which no cache holds: 2^27 values 58 us (62 with one), 2^26 25.8 (25.5),
// 2^23 5.2 (4.9). f32 takes one (2^27 values 112 us, 137 with four), and so does packing (2^27 57 and 59, f32 105 and 112).
template <typename T>
hipError_t unpack(const unsigned char* codes, const unsigned char* scales, void* x, long vectors, hipStream_t stream) {
  if constexpr (sizeof(T) == 2)
    if (vectors >= 1l << 24) return launch_unpack<T, 4>(codes, scales, x, vectors, stream);
  return launch_unpack<T, 1>(codes, scales, x, vectors, stream);
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
