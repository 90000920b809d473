// Attention of new tokens over a paged cache on gfx950 with f32 arithmetic throughout:
//   out[t, hq, :] = sum_j softmax_j(scale * q[t, hq] . k_j) v_j over the keys j of t's sequence that it may see
// (all of them, or, causal, those up to its own position), k and v rows of key head hq / group.
//
// Work: a workgroup takes 16 RB rows (new token x query head of one key head, so that the heads that share keys share
// their loads) and one range of keys; its four waves take the range's blocks of 32 keys in turn and join their
// online softmaxes at the end. S^T = K Q^T and O^T += V^T P^T run on v_mfma_f32_16x16x4: a lane's 16-byte load of a
// key row is the A operand of four products whose reduction index is permuted alike for q, and a 16-byte load of a
// value row is A of four products with the output columns permuted, so K and V go from memory to the matrix units
// without passing LDS, and P stays in the lane that made it.
//
// What bounds it: the f32 matrix rate (64 flops a cycle and SIMD) where many rows share the keys, else the bytes of
// K and V. 16 rows use each value loaded for 8 flops a byte, twice what L1 would need to keep up.
#include "paged.hpp"

namespace samhip {

namespace {

__device__ __forceinline__ f32x4 mma4(float a, float b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

// Four consecutive elements as f32.
__device__ __forceinline__ f32x4 load4(const float* p) { return *reinterpret_cast<const f32x4*>(p); }
__device__ __forceinline__ f32x4 load4(const e4m3* p) {
  typedef float f2 __attribute__((ext_vector_type(2)));
  const int c = *reinterpret_cast<const int*>(p);
  const f2 a = __builtin_amdgcn_cvt_pk_f32_fp8(c, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(c, true);
  return f32x4{a[0], a[1], b[0], b[1]};
}

template <typename T, typename C, int DP, int RB>
__global__ __launch_bounds__(256, DP * RB <= 128 ? 2 : 1) void paged_f32_kernel(PagedParams p) {
  constexpr int NC = DP / 16, ND = DP / 64, TR = 16 * RB;
  constexpr bool kScaled = __is_same(C, e4m3);
  __shared__ float sm_m[2][TR], sm_l[2][TR];
  extern __shared__ __attribute__((aligned(16))) float sm_o[];  // [2][RB][DP / 4 * 64]
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int n = lane & 15, g = lane >> 4;
  const int d = p.c.d;
  if (p.zero_rest) paged_zero_rest<T>(p);
  const PagedWork w = paged_work(p);
  const int rows = w.lq * p.group;
  const C* kp = reinterpret_cast<const C*>(p.c.k);
  const C* vp = reinterpret_cast<const C*>(p.c.v);

  for (int rt = w.tile; (long)rt * TR < rows; rt += p.rtiles) {
    long qoff[RB];
    int limit[RB], tok[RB], head[RB];
    f32x4 qf[RB][NC];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      const int r = min(rt * TR + 16 * rb + n, rows - 1);
      const int t = (int)divide_magic(r, p.gmagic, p.gshift);
      tok[rb] = w.s0 + t;
      head[rb] = w.head * p.group + (r - t * p.group);
      limit[rb] = p.causal ? max(0, min(w.len, w.len - w.lq + t + 1)) : w.len;
      qoff[rb] = tok[rb] * p.sq[0] + head[rb] * p.sq[1];
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int col = 16 * c + 4 * g;
        qf[rb][c] = col < d ? load4(reinterpret_cast<const T*>(p.q) + qoff[rb] + col) : f32x4{};
      }
    }
    // the keys that the tile's last row sees; this split's blocks of 32 of them
    const int tlast = (int)divide_magic(min((rt + 1) * TR, rows) - 1, p.gmagic, p.gshift);
    const int most = p.causal ? max(0, min(w.len, w.len - w.lq + tlast + 1)) : w.len;
    const int tfirst = (int)divide_magic(rt * TR, p.gmagic, p.gshift);
    const int least = p.causal ? max(0, min(w.len, w.len - w.lq + tfirst + 1)) : w.len;
    const int blocks = (most + 31) >> 5, per = paged_share(blocks, p.per, p.nsplit);
    const int b0 = min(blocks, w.split * per), b1 = min(blocks, b0 + per);
    const bool direct = blocks <= per;  // one split has all keys: it writes the result itself
    if (direct && w.split > 0) continue;

    float m[RB], l[RB];
    f32x4 o[RB][4 * ND];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      m[rb] = -INFINITY;
      l[rb] = 0.f;
#pragma unroll
      for (int i = 0; i < 4 * ND; ++i) o[rb][i] = f32x4{};
    }
    for (int blk = b0 + wave; blk < b1; blk += 4) {
      const int key0 = 32 * blk;
      const bool part = key0 + 32 > least;
      const int row = paged_row(p.c, w.b, w.head, key0 + (lane & 31), most);  // lane l looks key l % 32 up
      const unsigned there = (unsigned)__builtin_amdgcn_ballot_w64(row >= 0);
      float ks = 1.f, vs = 1.f;
      if (kScaled && row >= 0) {
        ks = pow2_of(p.c.ks[row]);
        vs = pow2_of(p.c.vs[row]);
      }
      f32x4 s[RB][2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const long kr = __shfl(row, 16 * i + n);
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) s[rb][i] = f32x4{};
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const int col = 16 * c + 4 * g;
          const f32x4 a = kr >= 0 && col < d ? load4(kp + kr * d + col) : f32x4{};
#pragma unroll
          for (int rb = 0; rb < RB; ++rb)
#pragma unroll
            for (int j = 0; j < 4; ++j) s[rb][i] = mma4(a[j], qf[rb][c][j], s[rb][i]);
        }
      }
      // s[rb][i][e]: key key0 + 16 i + 4 g + e, row 16 rb + n
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) {
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int kk = 16 * i + 4 * g + e;
            const bool sees = key0 + kk < limit[rb] && (there >> kk & 1);
            const float f = kScaled ? __shfl(ks, kk) : 1.f;
            s[rb][i][e] = sees ? s[rb][i][e] * (p.sc * f) : -INFINITY;
            top = max_nc(top, s[rb][i][e]);
          }
        top = max_over_rows16(top);
        const float mn = fmaxf(m[rb], top);
        const float base = mn == -INFINITY ? 0.f : mn;
        const float alpha = exp2_fast(m[rb] - base);
        m[rb] = mn;
        l[rb] *= alpha;
#pragma unroll
        for (int i = 0; i < 4 * ND; ++i) o[rb][i] *= alpha;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            s[rb][i][e] = exp2_fast(s[rb][i][e] - base);
            l[rb] += s[rb][i][e];
          }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int kk = 16 * i + 4 * g + e;
          const long vr = __shfl(row, kk);
          const float f = kScaled ? __shfl(vs, kk) : 1.f;
#pragma unroll
          for (int q = 0; q < ND; ++q) {
            const int col = 64 * q + 4 * n;
            f32x4 a = vr >= 0 && col < d ? load4(vp + vr * d + col) : f32x4{};
            // a value that is not finite must not reach the rows that do not see its key (0 * inf = NaN): where the
            // block's keys are not seen by every row, such values are taken out, and the rows that see one get
            // inf for +inf, -inf for -inf and both for NaN, counted on the matrix unit
            bool odd = false;
            if (part) {
#pragma unroll
              for (int j = 0; j < 4; ++j) odd |= !(fabsf(a[j]) < INFINITY);
            }
            if (part && wave_any(odd)) {
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const float up = !(a[j] < INFINITY) ? 1.f : 0.f, down = !(a[j] > -INFINITY) ? 1.f : 0.f;
                a[j] = up + down > 0.f ? 0.f : a[j];
#pragma unroll
                for (int rb = 0; rb < RB; ++rb) {
                  const float sees = key0 + kk < limit[rb] ? 1.f : 0.f;
                  const f32x4 hi = mma4(up, sees, f32x4{}), lo = mma4(down, sees, f32x4{});
#pragma unroll
                  for (int k = 0; k < 4; ++k)
                    o[rb][4 * q + j][k] += (hi[k] > 0.f ? INFINITY : 0.f) + (lo[k] > 0.f ? -INFINITY : 0.f);
                }
              }
            }
#pragma unroll
            for (int rb = 0; rb < RB; ++rb)
#pragma unroll
              for (int j = 0; j < 4; ++j) o[rb][4 * q + j] = mma4(a[j], s[rb][i][e] * f, o[rb][4 * q + j]);
          }
        }
    }
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) l[rb] = sum_over_rows16(l[rb]);

    // join the waves: 2 and 3 into 0 and 1, then 1 into 0
    for (int half = 2; half >= 1; half /= 2) {
      __syncthreads();
      if (wave >= half && wave < 2 * half) {
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
          if (g == 0) {
            sm_m[wave - half][16 * rb + n] = m[rb];
            sm_l[wave - half][16 * rb + n] = l[rb];
          }
#pragma unroll
          for (int i = 0; i < 4 * ND; ++i)
            *reinterpret_cast<f32x4*>(sm_o + (((wave - half) * RB + rb) * 4 * ND + i) * 256 + 4 * lane) = o[rb][i];
        }
      }
      __syncthreads();
      if (wave < half) {
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
          const float mo = sm_m[wave][16 * rb + n], mn = fmaxf(m[rb], mo);
          const float base = mn == -INFINITY ? 0.f : mn;
          const float a = exp2_fast(m[rb] - base), c = exp2_fast(mo - base);
          l[rb] = l[rb] * a + sm_l[wave][16 * rb + n] * c;
          m[rb] = mn;
#pragma unroll
          for (int i = 0; i < 4 * ND; ++i)
            o[rb][i] = o[rb][i] * a +
                       *reinterpret_cast<const f32x4*>(sm_o + ((wave * RB + rb) * 4 * ND + i) * 256 + 4 * lane) * c;
        }
      }
    }
    if (wave == 0) {
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) {
        if (rt * TR + 16 * rb + n >= rows) continue;
        const long row = ((long)w.split * p.tokens + tok[rb]) * p.heads + head[rb];
        if (p.nsplit > 1 && g == 0)
          *reinterpret_cast<float2*>(p.ml + 2 * row) = direct ? float2{0.f, -1.f} : float2{m[rb], l[rb]};
        if (direct) {
          const float inv = l[rb] == 0.f ? 0.f : 1.f / l[rb];  // a row that sees no key is 0
          T* orow = reinterpret_cast<T*>(p.out) + tok[rb] * p.so[0] + head[rb] * p.so[1];
#pragma unroll
          for (int q = 0; q < ND; ++q)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int col = 64 * q + 16 * g + 4 * e;
              if (col >= d) continue;
              typename Vec<T>::x4 x;
#pragma unroll
              for (int j = 0; j < 4; ++j) x[j] = from_f32<T>(f32_result(o[rb][4 * q + j][e] * inv));
              *reinterpret_cast<typename Vec<T>::x4*>(orow + col) = x;
            }
        } else if (b0 < b1) {
#pragma unroll
          for (int q = 0; q < ND; ++q)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int col = 64 * q + 16 * g + 4 * e;
              if (col < d)
                *reinterpret_cast<f32x4*>(p.opart + row * d + col) =
                    f32x4{o[rb][4 * q][e], o[rb][4 * q + 1][e], o[rb][4 * q + 2][e], o[rb][4 * q + 3][e]};
            }
        }
      }
    }
    __syncthreads();
  }
}

template <typename T, typename C, int DP, int RB> hipError_t launch_f32(const PagedParams& p, hipStream_t stream) {
  constexpr int lds = 2 * RB * (DP / 4) * 64 * 4;
  static_assert(lds <= 64 << 10, "the joining buffer");
  const long blocks = (long)p.rtiles * p.nsplit * p.c.heads * p.c.batch;
  hipLaunchKernelGGL((paged_f32_kernel<T, C, DP, RB>), dim3((unsigned)blocks), dim3(256), lds, stream, p);
  return hipGetLastError();
}
template <typename T, typename C> hipError_t by_size(const PagedParams& p, int rows, hipStream_t stream) {
  const int d = p.c.d;
  if (rows == 16)
    return d <= 64 ? launch_f32<T, C, 64, 1>(p, stream)
                   : d <= 128 ? launch_f32<T, C, 128, 1>(p, stream) : launch_f32<T, C, 256, 1>(p, stream);
  return d <= 64 ? launch_f32<T, C, 64, 2>(p, stream) : launch_f32<T, C, 128, 2>(p, stream);
}

}  // namespace

hipError_t paged_f32(int cache_dtype, const PagedParams& p, int rows, hipStream_t stream) {
  return cache_dtype == kE4M3 ? by_size<float, e4m3>(p, rows, stream) : by_size<float, float>(p, rows, stream);
}

}  // namespace samhip
