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
// A weight is exp2((score - maximum) * scale): exact in the difference, so that scores of any size keep their order
// (score * scale - maximum * scale, one instruction less, rounds the latter and overflows from 2^31 on; 387 us below at 128).
//
// What bounds it: the f32 matrix rate (64 flops a cycle and SIMD) where many rows share the keys, else the bytes of
// K and V. 16 rows use each value loaded for 8 flops a byte, twice what L1 would need to keep up. 2048 rows over 4096 keys,
// 8 heads: head dim 64 191 us (90 TFLOP/s), 128 396 (87; a large library product 153), 256 with 4 heads 520 (66); a step of 32
// sequences of 4096 keys, 8 key heads of 128, 210 (5.1 TB/s); of 8192 keys from e2m1 pages 201 (e4m3 216), which the products
// bound.
#include "lds_dma.hpp"
#include "paged.hpp"

namespace samhip {

namespace {

__device__ __forceinline__ f32x4 mma4(float a, float b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

// Four elements of a cache row as they lie there, and as f32 (times their row's scale).
template <typename C> struct Raw4 {
  typedef f32x4 t;
};
template <> struct Raw4<e4m3> {
  typedef int t;
};
template <> struct Raw4<e2m1> {
  typedef unsigned short t;
};
__device__ __forceinline__ f32x4 widen(f32x4 x, float) { return x; }
__device__ __forceinline__ f32x4 widen(int c, float s) {
  typedef float f2 __attribute__((ext_vector_type(2)));
  const f2 a = __builtin_amdgcn_cvt_pk_f32_fp8(c, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(c, true);
  return f32x4{a[0] * s, a[1] * s, b[0] * s, b[1] * s};
}

__device__ __forceinline__ f32x4 widen(unsigned short c, float s) {
  const f32x2 a = mx_decode2_f32<0>(c, s), b = mx_decode2_f32<1>(c, s);
  return f32x4{a[0], a[1], b[0], b[1]};
}
// The low or the high four codes of a word.
__device__ __forceinline__ f32x4 widen_half(unsigned w, bool high, float s) {
  const f32x2 a = high ? mx_decode2_f32<2>(w, s) : mx_decode2_f32<0>(w, s), b = high ? mx_decode2_f32<3>(w, s) : mx_decode2_f32<1>(w, s);
  return f32x4{a[0], a[1], b[0], b[1]};
}

template <typename C, int DP, int RB>
__global__ __launch_bounds__(256, DP * RB <= 64 ? 2 : 1) void paged_f32_kernel(PagedParams p) {
  constexpr int NC = DP / 16, ND = (DP + 63) / 64, TR = 16 * RB;
  constexpr bool kMx = __is_same(C, e2m1), kScaled = __is_same(C, e4m3);
  typedef typename Raw4<C>::t Raw;
  __shared__ float sm_m[2][TR], sm_l[2][TR];
  extern __shared__ __attribute__((aligned(16))) float sm_o[];  // [2][RB][4 ND][256]
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int d = p.c.d;
  if (p.zero_rest) paged_zero_rest<float>(p);
  const PagedWork w = paged_work(p);
  const int rows = w.lq * p.group;
  const C* kp = reinterpret_cast<const C*>(p.c.k);
  const C* vp = reinterpret_cast<const C*>(p.c.v);

  for (int rt = w.tile; (long)rt * TR < rows; rt += p.rtiles) {
    // hidden from the optimiser, which would keep every address derived from the lane in a register across tiles
    const int lane = (int)opaque(threadIdx.x & 63), n = lane & 15, g = lane >> 4;
    int limit[RB], tok[RB], head[RB];
    f32x4 qf[RB][NC];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      const int r = min(rt * TR + 16 * rb + n, rows - 1);
      const int t = (int)divide_magic(r, p.gmagic, p.gshift);
      tok[rb] = w.s0 + t;
      head[rb] = w.head * p.group + (r - t * p.group);
      limit[rb] = paged_keys(w, p.causal, t);
      const float* qr = reinterpret_cast<const float*>(p.q) + tok[rb] * p.sq[0] + head[rb] * p.sq[1];
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int col = kMx ? DP / 4 * g + 4 * c : 16 * c + 4 * g;
        qf[rb][c] = col < d ? *reinterpret_cast<const f32x4*>(qr + col) : f32x4{};
      }
    }
    // the keys that the tile's first and last row see; this split's blocks of 32 of them
    const int tfirst = (int)divide_magic(rt * TR, p.gmagic, p.gshift);
    const int tlast = (int)divide_magic(min((rt + 1) * TR, rows) - 1, p.gmagic, p.gshift);
    const int least = paged_keys(w, p.causal, tfirst);
    const int most = paged_keys(w, p.causal, tlast);
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
    // lane l looks key l % 32 of a block up; rows that are not there read row 0 and are masked (K) or cleared (V)
    auto entry_of = [&](int blk) { return paged_entry(p.c, w.b, 32 * min(blk, b1 - 1) + (lane & 31), most); };
    const unsigned at_n = opaque(4 * n), at_g = opaque(16 * g);  // lanes n and 4 g, as bpermute addresses
    auto from_n = [&](int i, int v) { return __builtin_amdgcn_ds_bpermute((int)at_n + 64 * i, v); };
    auto from_key = [&](int j, int v) {  // the lane whose own key is 16 (j / 4) + 4 g + j % 4
      return __builtin_amdgcn_ds_bpermute((int)at_g + 64 * (j >> 2) + 4 * (j & 3), v);
    };
    Raw kx[2][kMx ? 1 : NC], vx[8][ND];
    unsigned char ksx = 127, vsx = 127;
    // e2m1: a lane's words of a key row lie side by side, DP / 4 columns, of one or two blocks (a word each at 96), which q's
    // columns follow; the scales of every other of its own key's value blocks (lanes 0 .. 31 the even ones)
    constexpr int KW = DP / 32, KSC = DP == 96 ? 3 : DP <= 128 ? 1 : 2;
    unsigned kw[2][KW];
    unsigned char kmx[2][KSC], vmx[ND];
    const int G = d / kMxBlock;
    auto load_k = [&](int row) {
      if constexpr (kScaled) ksx = p.c.ks[max(row, 0)];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const long r = max(from_n(i, row), 0);
        const C* kr = held_at(kp, r * d);
        if constexpr (kMx) {
          constexpr int KL = KW % 4 == 0 ? 4 : KW == 2 ? 2 : 1;  // words of a load
#pragma unroll
          for (int w = 0; w < KW; w += KL) {
            const C* at = held_at(kr, min(DP / 4 * g + 8 * w, d - 8 * KL));
            if constexpr (KL == 4)
              *reinterpret_cast<u32x4*>(&kw[i][w]) = *reinterpret_cast<const u32x4*>(at);
            else if constexpr (KL == 2)
              *reinterpret_cast<u32x2*>(&kw[i][w]) = *reinterpret_cast<const u32x2*>(at);
            else
              kw[i][w] = *reinterpret_cast<const unsigned*>(at);
          }
#pragma unroll
          for (int b = 0; b < KSC; ++b) kmx[i][b] = p.c.ks[r * G + min((DP / 4 * g + (DP == 96 ? 8 : 32) * b) / kMxBlock, G - 1)];
        } else {
#pragma unroll
          for (int c = 0; c < NC; ++c) kx[i][c] = *reinterpret_cast<const Raw*>(held_at(kr, min(16 * c + 4 * g, d - 4)));
        }
      }
    };
    auto load_v = [&](int row) {
      if constexpr (kScaled) vsx = p.c.vs[max(row, 0)];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const C* vr = held_at(vp, (long)max(from_key(j, row), 0) * d);
#pragma unroll
        for (int q = 0; q < ND; ++q) vx[j][q] = *reinterpret_cast<const Raw*>(held_at(vr, min(64 * q + 4 * n, d - 4)));
      }
      if constexpr (kMx) {
#pragma unroll
        for (int q = 0; q < ND; ++q) vmx[q] = p.c.vs[(long)max(row, 0) * G + min(2 * q + (lane >> 5), G - 1)];
      }
    };
    // Table entries two blocks ahead, K one, V while its block's scores are made
    int row = -1;
    PagedEntry coming = {-1, -1};
    if (b0 + wave < b1) {
      const PagedEntry first = entry_of(b0 + wave);
      coming = entry_of(b0 + wave + 4);
      row = paged_row(p.c, first, w.head);
      load_k(row);
    }
    // Q is here: told to the compiler, whose own wait for it would stand in the loop, behind the next block's loads
    __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
    for (int blk = b0 + wave; blk < b1; blk += 4) {
      const int key0 = 32 * blk;
      const int next = paged_row(p.c, coming, w.head);
      coming = entry_of(blk + 8);
      load_v(row);
      const unsigned there = (unsigned)__builtin_amdgcn_ballot_w64(row >= 0);
      const bool part = key0 + 32 > least || there != 0xffffffffu;
      const unsigned mine = there >> (4 * g);  // bit 16 i + e: the lane's key 16 i + 4 g + e
      f32x4 s[RB][2];
      const float kso = kScaled ? pow2_of(ksx) : 1.f;
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) s[rb][0] = s[rb][1] = f32x4{};
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float f = 1.f;
        if constexpr (kScaled) f = __int_as_float(from_n(i, __float_as_int(kso)));
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          f32x4 a;
          if constexpr (kMx)
            a = widen_half(kw[i][c / 2], c % 2, mx_scale(kmx[i][DP == 96 ? c / 2 : c / 8 % KSC]));
          else
            a = widen(kx[i][c], f);
          if (kMx ? DP / 4 * g + 4 * c >= d : 16 * c + 16 > d && 16 * c + 4 * g >= d) a = f32x4{};
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) s[rb][i] = mma4(a[j], qf[rb][c][j], s[rb][i]);
        }
      }
      load_k(next);  // after the last block the range's last again: under a condition, V would wait for it too
      // s[rb][i][e]: key key0 + 16 i + 4 g + e, row 16 rb + n
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) {
        if (part) {
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int kk = 16 * i + e;
              s[rb][i][e] = kk < limit[rb] - key0 - 4 * g && (mine >> kk & 1) ? s[rb][i][e] : -INFINITY;
            }
        }
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) top = max_nc(top, s[rb][i][e]);
        const float mn = fmaxf(m[rb], max_over_rows16(top));
        const float base = mn == -INFINITY ? 0.f : mn;
        const float alpha = exp2_fast((m[rb] - base) * p.sc);
        m[rb] = mn;
        l[rb] *= alpha;
#pragma unroll
        for (int i = 0; i < 4 * ND; ++i) o[rb][i] *= alpha;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            s[rb][i][e] = exp2_fast((s[rb][i][e] - base) * p.sc);
            l[rb] += s[rb][i][e];
          }
      }
      bool odd = false;
      const float vso = kScaled ? pow2_of(vsx) : 1.f;
      float vs[8];
      if constexpr (kScaled) {
#pragma unroll
        for (int j = 0; j < 8; ++j) vs[j] = __int_as_float(from_key(j, __float_as_int(vso)));
      }
      unsigned vm[8];
      if constexpr (kMx) {
        unsigned vmo = 0;
#pragma unroll
        for (int q = 0; q < ND; ++q) vmo |= (unsigned)vmx[q] << (8 * q);
#pragma unroll
        for (int j = 0; j < 8; ++j) vm[j] = (unsigned)__builtin_amdgcn_ds_bpermute((int)at_g + 128 * (n >> 3) + 64 * (j >> 2) + 4 * (j & 3), (int)vmo);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int q = 0; q < ND; ++q) {
          f32x4 a = widen(vx[j][q], kMx ? mx_scale(vm[j] >> (8 * q) & 255) : kScaled ? vs[j] : 1.f);
          if (part) {  // rows that are not there hold anything; values that are not finite go apart
            const bool ok = mine >> (16 * (j >> 2) + (j & 3)) & 1;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const bool fin = fabsf(a[i]) < INFINITY;
              odd |= ok && !fin;
              a[i] = ok && fin ? a[i] : 0.f;
            }
          }
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) o[rb][4 * q + i] = mma4(a[i], s[rb][j >> 2][j & 3], o[rb][4 * q + i]);
        }
      if (wave_any(odd)) {
        // A value that is not finite must not reach the rows that do not see its key (0 * inf = NaN): it was taken out
        // above, and the rows that see it add it here
        for (int kk = 0; kk < 32; ++kk) {
          if (!(there >> kk & 1)) continue;
          const int kr = __shfl(row, kk);
          const float f = kScaled ? pow2_of(p.c.vs[kr]) : 1.f;
#pragma unroll
          for (int q = 0; q < ND; ++q)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int col = 64 * q + 16 * g + 4 * e;
              if (col < d) {
                const float fc = kMx ? mx_scale(p.c.vs[(long)kr * G + col / kMxBlock]) : f;
                const f32x4 x = widen(*reinterpret_cast<const Raw*>(held_at(vp, (long)kr * d + col)), fc);
#pragma unroll
                for (int rb = 0; rb < RB; ++rb)
#pragma unroll
                  for (int j = 0; j < 4; ++j)
                    o[rb][4 * q + j][e] += key0 + kk < limit[rb] && !(fabsf(x[j]) < INFINITY) ? x[j] : 0.f;
              }
            }
        }
      }
      row = next;
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
          const float a = exp2_fast((m[rb] - base) * p.sc), c = exp2_fast((mo - base) * p.sc);
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
          *reinterpret_cast<float2*>(p.ml + 2 * row) = direct ? float2{0.f, -1.f} : float2{m[rb] * p.sc, l[rb]};
        if (direct) {
          const float inv = l[rb] == 0.f ? 0.f : 1.f / l[rb];  // a row that sees no key is 0
          float* orow = reinterpret_cast<float*>(p.out) + tok[rb] * p.so[0] + head[rb] * p.so[1];
#pragma unroll
          for (int q = 0; q < ND; ++q)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int col = 64 * q + 16 * g + 4 * e;
              if (col >= d) continue;
              f32x4 x;
#pragma unroll
              for (int j = 0; j < 4; ++j) x[j] = o[rb][4 * q + j][e] * inv;
              *reinterpret_cast<f32x4*>(orow + col) = x;
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

template <typename C, int DP, int RB> hipError_t launch_f32(const PagedParams& p, hipStream_t stream) {
  constexpr int lds = 2 * RB * 4 * ((DP + 63) / 64) * 256 * 4;
  static_assert(lds <= 64 << 10, "the joining buffer");
  const long blocks = (long)p.rtiles * p.nsplit * p.c.heads * p.c.batch;
  hipLaunchKernelGGL((paged_f32_kernel<C, DP, RB>), dim3((unsigned)blocks), dim3(256), lds, stream, p);
  return hipGetLastError();
}
template <typename C> hipError_t by_size(const PagedParams& p, int rows, hipStream_t stream) {
  const int d = p.c.d;
  if (rows == 16)
    return d <= 64 ? launch_f32<C, 64, 1>(p, stream)
                   : d <= 128 ? launch_f32<C, 128, 1>(p, stream) : launch_f32<C, 256, 1>(p, stream);
  return d <= 64 ? launch_f32<C, 64, 2>(p, stream)
                 : d <= 96 ? launch_f32<C, 96, 2>(p, stream) : launch_f32<C, 128, 2>(p, stream);
}

}  // namespace

hipError_t paged_f32(int cache_dtype, const PagedParams& p, int rows, hipStream_t stream) {
  if (cache_dtype == kE2M1) return by_size<e2m1>(p, rows, stream);
  return cache_dtype == kE4M3 ? by_size<e4m3>(p, rows, stream) : by_size<float>(p, rows, stream);
}

}  // namespace samhip
