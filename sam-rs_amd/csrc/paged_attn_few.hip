// Paged attention on gfx950 for few rows a key head (a decoding step, a short chunk), f16 / bf16 queries over pages of
// their own type or of e4m3.
//
// What bounds it: the bytes of K and V, each used for 4 flops a row. So nothing stands between memory and the matrix
// units: a wave takes blocks of 32 keys of its workgroup's range, loads their K and V rows straight into registers, the
// next block's K while it weighs this one's V and the next V during the next scores, and passes neither through LDS.
//   S^T = K Q^T on v_mfma_f32_16x16x32: a lane's 16 bytes (8 codes) of key row n are an A operand as they are.
//   O^T += V^T P^T: a lane loads the same few columns of 8 keys, whose 16-bit pairs v_perm_b32 transposes in registers
//   into A operands (the output's columns come out permuted, which the store undoes); P stays where S^T left it, since
//   the reduction index is permuted alike: element j of lane group g is key 16 (j / 4) + 4 g + j % 4.
// e4m3 codes become 16-bit values with their row's scale in one conversion, exactly (in f16, values below 2^-14 to
// f16's subnormal step). Softmax statistics and sums are f32. f16 P is rounded to f16 and its sum taken over the rounded
// values, all of it times 2^15, which O / l cancels: weights keep f16's 11 bits down to 2^-29 of the largest, so that
// thousands of keys far below one that dominates are not lost (each is off by 2^-40 of it at most). The exponent is taken of
// (score - maximum) * scale, so that scores of any size keep P in f16's range. bf16 P goes as
// hi + lo, which leaves 2^-16 of it (one bf16 term would leave 2^-8, as much as the output's own rounding).
//
// The four waves of a workgroup join at its end, the key ranges of a sequence in paged_combine_kernel.
//
// Measured, 32 sequences of 8192 keys, 8 key heads of 128, one token of 4 query heads a key head: f16 pages 187 us (5.7
// TB/s), e4m3 pages 107 with f16 queries and 123 with bf16 (5.0 and 4.4; not for their instructions: a fifth fewer took as
// long). 64-key blocks of e4m3 were no faster.
#include "lds_dma.hpp"
#include "paged.hpp"

namespace samhip {

namespace {

template <int BYTES> struct Raw;
template <> struct Raw<4> {
  typedef unsigned t;
};
template <> struct Raw<8> {
  typedef u32x2 t;
};
template <> struct Raw<16> {
  typedef u32x4 t;
};

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

// Workgroups a CU: as many as registers allow with a block of K and one of V in flight. Three for e4m3 at head dim 128
// (131 us for the bf16 call above with eight splits, 137 with two).
template <typename T, typename C, int DP, int RB>
__global__ __launch_bounds__(256, DP * RB > 128 ? 1 : DP == 128 && !__is_same(C, e4m3) ? 2 : 3) void paged_few_kernel(PagedParams p) {
  typedef typename Vec<T>::x8 X8;
  constexpr bool kCoded = __is_same(C, e4m3), kSplitP = __is_same(T, bf16);
  constexpr float kLift = kSplitP ? 0.f : 15.f;  // P is lifted by 2^kLift
  constexpr int TR = 16 * RB, NK = DP / 32;
  constexpr int CW = DP >= 128 ? 8 : DP / 16, NV = DP / (16 * CW);  // columns of a value row that a lane takes at once
  typedef typename Raw<8 * (int)sizeof(C)>::t KRaw;
  typedef typename Raw<CW * (int)sizeof(C)>::t VRaw;
  __shared__ float sm_m[2][TR], sm_l[2][TR];
  __shared__ __attribute__((aligned(16))) float sm_o[2][RB * DP / 16][256];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int d = p.c.d;
  if (p.zero_rest) paged_zero_rest<T>(p);
  const PagedWork w = paged_work(p);
  const int rows = w.lq * p.group;
  const C* kp = reinterpret_cast<const C*>(p.c.k);
  const C* vp = reinterpret_cast<const C*>(p.c.v);

  for (int rt = w.tile; (long)rt * TR < rows; rt += p.rtiles) {
    // hidden from the optimiser, which would keep every address derived from the lane in a register across tiles
    const int lane = (int)opaque(threadIdx.x & 63), n = lane & 15, g = lane >> 4;
    const int tfirst = (int)divide_magic(rt * TR, p.gmagic, p.gshift);
    const int tlast = (int)divide_magic(min((rt + 1) * TR, rows) - 1, p.gmagic, p.gshift);
    const int most = paged_keys(w, p.causal, tlast);
    const int least = paged_keys(w, p.causal, tfirst);
    // this split's blocks of 32 keys: ranges of the hint's longest sequence, longer ones where that was too short
    const int blocks = (most + 31) >> 5, per = paged_share(blocks, p.per, p.nsplit);
    const int b0 = min(blocks, w.split * per), b1 = min(blocks, b0 + per);
    const bool direct = blocks <= per;  // one split has all keys: it writes the result itself
    if (direct && w.split > 0) continue;

    int limit[RB];
    X8 qf[RB][NK];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      const int r = min(rt * TR + 16 * rb + n, rows - 1);
      const int t = (int)divide_magic(r, p.gmagic, p.gshift);
      limit[rb] = paged_keys(w, p.causal, t);
      const T* qr = reinterpret_cast<const T*>(p.q) + (w.s0 + t) * p.sq[0] + (w.head * p.group + r - t * p.group) * p.sq[1];
#pragma unroll
      for (int c = 0; c < NK; ++c) {
        const int col = 32 * c + 8 * g;
        qf[rb][c] = col < d ? *reinterpret_cast<const X8*>(qr + col) : X8{};
      }
    }

    float m[RB], l[RB];
    f32x4 o[RB][DP / 16];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      m[rb] = -INFINITY;
      l[rb] = 0.f;
#pragma unroll
      for (int i = 0; i < DP / 16; ++i) o[rb][i] = f32x4{};
    }

    // a block's rows: lane l looks key l % 32 up. Rows that are not there read row 0 and are masked (K) or cleared (V).
    const unsigned at_n = opaque(4 * n), at_g = opaque(16 * g);  // lanes n and 4 g, as bpermute addresses
    auto from_n = [&](int i, int v) { return __builtin_amdgcn_ds_bpermute((int)at_n + 64 * i, v); };
    auto from_key = [&](int j, int v) {  // the lane whose own key is element j of group g
      return __builtin_amdgcn_ds_bpermute((int)at_g + 64 * (j >> 2) + 4 * (j & 3), v);
    };
    auto entry_of = [&](int blk) { return paged_entry(p.c, w.b, 32 * min(blk, b1 - 1) + (lane & 31), most); };
    KRaw kx[2][NK];
    VRaw vx[8][NV];
    unsigned char ksx = 127, vsx = 127;  // scales of the lane's own key
    auto load_k = [&](int row) {
      if constexpr (kCoded) ksx = p.c.ks[max(row, 0)];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const C* kr = kp + (long)max(from_n(i, row), 0) * d;
#pragma unroll
        for (int c = 0; c < NK; ++c) kx[i][c] = *reinterpret_cast<const KRaw*>(kr + min(32 * c + 8 * g, d - 8));
      }
    };
    auto load_v = [&](int row) {
      if constexpr (kCoded) vsx = p.c.vs[max(row, 0)];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const C* vr = vp + (long)max(from_key(j, row), 0) * d;
#pragma unroll
        for (int q = 0; q < NV; ++q) vx[j][q] = *reinterpret_cast<const VRaw*>(vr + min(CW * (16 * q + n), d - CW));
      }
    };

    // Table entries two blocks ahead, K and V one: a wait for a load waits for those before it too, so the entries go
    // ahead of the rows that they are not needed for. After its last block a wave loads the range's last again: loads under
    // a condition would have the next scores wait for V too, as the compiler counts what is in flight on the shorter path.
    int row = -1;
    PagedEntry coming = {-1, -1};
    if (b0 + wave < b1) {
      const PagedEntry first = entry_of(b0 + wave);
      coming = entry_of(b0 + wave + 4);
      row = paged_row(p.c, first, w.head);
      load_k(row);
      load_v(row);
    }
    // Q is here: told to the compiler, whose own wait for it would stand in the loop, behind the next block's loads
    __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
    for (int blk = b0 + wave; blk < b1; blk += 4) {
      const int key0 = 32 * blk;
      const int next = paged_row(p.c, coming, w.head);
      coming = entry_of(blk + 8);
      const unsigned there = (unsigned)__builtin_amdgcn_ballot_w64(row >= 0);
      f32x4 s[RB][2];
      const float kso = kCoded ? pow2_of(ksx) : 1.f, vso = kCoded ? pow2_of(vsx) : 1.f;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float ks = 1.f;
        if constexpr (kCoded) ks = __int_as_float(from_n(i, __float_as_int(kso)));
#pragma unroll
        for (int c = 0; c < NK; ++c) {
          u32x4 a;
          if constexpr (kCoded)
            a = u32x4{decode2<T, false>(kx[i][c][0], ks), decode2<T, true>(kx[i][c][0], ks),
                      decode2<T, false>(kx[i][c][1], ks), decode2<T, true>(kx[i][c][1], ks)};
          else
            a = kx[i][c];
          if (32 * c + 32 > d && 32 * c + 8 * g >= d) a = u32x4{};
#pragma unroll
          for (int rb = 0; rb < RB; ++rb)
            s[rb][i] = mma16(__builtin_bit_cast(X8, a), qf[rb][c], c == 0 ? f32x4{} : s[rb][i]);
        }
      }
      // s[rb][i][e]: key key0 + 16 i + 4 g + e, row 16 rb + n
      load_k(next);  // in flight while this block's V is weighed
      const bool part = key0 + 32 > least || there != 0xffffffffu;
      const unsigned mine = there >> (4 * g);  // bit 16 i + e: the lane's key 16 i + 4 g + e
      X8 b[RB], blo[RB];
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) {
        float top = -INFINITY;
        if (part) {
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int kk = 16 * i + e;
              s[rb][i][e] = kk < limit[rb] - key0 - 4 * g && (mine >> kk & 1) ? s[rb][i][e] : -INFINITY;
            }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) top = max_nc(top, s[rb][i][e]);
        const float m_new = fmaxf(m[rb], max_over_rows16(top));
        const float base = m_new == -INFINITY ? 0.f : m_new;
        const float alpha = exp2_fast((m[rb] - base) * p.sc);
        m[rb] = m_new;
        l[rb] *= alpha;
#pragma unroll
        for (int i = 0; i < DP / 16; ++i) o[rb][i] *= alpha;
        float pv[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          pv[j] = exp2_fast(fmaf(s[rb][j >> 2][j & 3] - base, p.sc, kLift));
        }
        if constexpr (kSplitP) {
#pragma unroll
          for (int j = 0; j < 8; ++j) l[rb] += pv[j];
          split_hi_lo(pv, b[rb], blo[rb]);
        } else {
          b[rb] = pack8(pv, (X8*)nullptr);
#pragma unroll
          for (int j = 0; j < 8; j += 2)
            l[rb] = __builtin_amdgcn_fdot2(f16x2{b[rb][j], b[rb][j + 1]}, f16x2{(f16)1.f, (f16)1.f}, l[rb], false);
        }
      }
      unsigned odd = 0;
      float vs[8];
      if constexpr (kCoded) {
#pragma unroll
        for (int j = 0; j < 8; ++j) vs[j] = __int_as_float(from_key(j, __float_as_int(vso)));
      }
#pragma unroll
      for (int q = 0; q < NV; ++q) {
        unsigned v[8][CW / 2];  // key j's columns, two to a register
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if constexpr (kCoded) {
#pragma unroll
            for (int h = 0; h < CW / 4; ++h) {
              unsigned word;
              if constexpr (CW == 8)
                word = vx[j][q][h];
              else
                word = vx[j][q];
              v[j][2 * h] = decode2<T, false>(word, vs[j]);
              v[j][2 * h + 1] = decode2<T, true>(word, vs[j]);
            }
          } else {
#pragma unroll
            for (int h = 0; h < CW / 2; ++h) v[j][h] = vx[j][q][h];
          }
          if (part) {  // rows that are not there hold anything; values that are not finite go apart
            const bool ok = mine >> (16 * (j >> 2) + (j & 3)) & 1;
#pragma unroll
            for (int h = 0; h < CW / 2; ++h) {
              const unsigned bad = not_finite2<T>(v[j][h]);
              v[j][h] = ok ? without2(v[j][h], bad) : 0u;
              odd |= ok ? bad : 0u;
            }
          }
        }
#pragma unroll
        for (int c = 0; c < CW; ++c) {
          u32x4 a;
#pragma unroll
          for (int j = 0; j < 4; ++j)  // keys 2 j and 2 j + 1 of column c
            a[j] = __builtin_amdgcn_perm(v[2 * j + 1][c >> 1], v[2 * j][c >> 1], c & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
          for (int rb = 0; rb < RB; ++rb) {
            f32x4& acc = o[rb][q * CW + c];
            acc = mma16(__builtin_bit_cast(X8, a), b[rb], acc);
            if constexpr (kSplitP) acc = mma16(__builtin_bit_cast(X8, a), blo[rb], acc);
          }
        }
      }
      if (wave_any(odd != 0)) {
        // A value that is not finite must not reach the rows that do not see its key (0 * inf = NaN): it was taken out
        // above, and the rows that see it add it here
        for (int kk = 0; kk < 32; ++kk) {
          if (!(there >> kk & 1)) continue;
          const int kr = __shfl(row, kk);
          const float s1 = kCoded ? pow2_of(p.c.vs[kr]) : 1.f;
#pragma unroll
          for (int q = 0; q < NV; ++q)
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
              for (int c = 0; c < CW; c += 4) {
                const int col = CW * (16 * q + 4 * g + e) + c;
                if (col < d) {
                  const f32x4 x = only_not_finite4<T>(vp + (long)kr * d + col, s1);
#pragma unroll
                  for (int rb = 0; rb < RB; ++rb)
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[rb][q * CW + c + i][e] += key0 + kk < limit[rb] ? x[i] : 0.f;
                }
              }
        }
      }
      load_v(next);
      row = next;
    }
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) l[rb] = sum_over_rows16(l[rb]);

    // join the waves: 2 and 3 into 0 and 1, then 1 into 0
#pragma unroll
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
          for (int i = 0; i < DP / 16; ++i)
            *reinterpret_cast<f32x4*>(&sm_o[wave - half][rb * (DP / 16) + i][4 * lane]) = o[rb][i];
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
          for (int i = 0; i < DP / 16; ++i)
            o[rb][i] = o[rb][i] * a + *reinterpret_cast<const f32x4*>(&sm_o[wave][rb * (DP / 16) + i][4 * lane]) * c;
        }
      }
    }
    if (wave == 0) {
      const int lane = (int)opaque(threadIdx.x & 63), n = lane & 15, g = lane >> 4;
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) {
        const int r = rt * TR + 16 * rb + n;
        if (r >= rows) continue;
        const int t = (int)divide_magic(r, p.gmagic, p.gshift);
        const long tok = w.s0 + t;
        const int hq = w.head * p.group + (r - t * p.group);
        const float inv = l[rb] == 0.f ? 0.f : 1.f / l[rb];  // a row that sees no key is 0
        const long part = (w.split * (long)p.tokens + tok) * p.heads + hq;
#pragma unroll
        for (int q = 0; q < NV; ++q)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int col = CW * (16 * q + 4 * g + e);  // o[q CW + c][e]: column col + c
            if (col >= d) continue;
            if (direct) {
              T* to = reinterpret_cast<T*>(p.out) + tok * p.so[0] + hq * p.so[1] + col;
#pragma unroll
              for (int c = 0; c < CW; c += 4) {
                typename Vec<T>::x4 y;
#pragma unroll
                for (int i = 0; i < 4; ++i) y[i] = from_f32<T>(f32_result(o[rb][q * CW + c + i][e] * inv));
                *reinterpret_cast<typename Vec<T>::x4*>(to + c) = y;
              }
            } else if (b0 < b1) {
              float* to = p.opart + part * d + col;
#pragma unroll
              for (int c = 0; c < CW; c += 4)
                *reinterpret_cast<f32x4*>(to + c) = f32x4{o[rb][q * CW + c][e], o[rb][q * CW + c + 1][e],
                                                          o[rb][q * CW + c + 2][e], o[rb][q * CW + c + 3][e]};
            }
          }
        if (p.nsplit > 1 && g == 0)
          *reinterpret_cast<float2*>(p.ml + 2 * part) = direct ? float2{0.f, -1.f} : float2{m[rb] * p.sc, l[rb]};
      }
    }
    __syncthreads();
  }
}

template <typename T, typename C, int DP, int RB> hipError_t launch_few(const PagedParams& p, hipStream_t stream) {
  const long blocks = (long)p.rtiles * p.nsplit * p.c.heads * p.c.batch;
  hipLaunchKernelGGL((paged_few_kernel<T, C, DP, RB>), dim3((unsigned)blocks), dim3(256), 0, stream, p);
  return hipGetLastError();
}
template <typename T, typename C> hipError_t by_size(const PagedParams& p, int rows, hipStream_t stream) {
  const int d = p.c.d;
  if (rows == 16)
    return d <= 64 ? launch_few<T, C, 64, 1>(p, stream)
                   : d <= 128 ? launch_few<T, C, 128, 1>(p, stream) : launch_few<T, C, 256, 1>(p, stream);
  return d <= 64 ? launch_few<T, C, 64, 2>(p, stream) : launch_few<T, C, 128, 2>(p, stream);
}

}  // namespace

hipError_t paged_few(int dtype, int cache_dtype, const PagedParams& p, int rows, hipStream_t stream) {
  if (dtype == kF16)
    return cache_dtype == kE4M3 ? by_size<f16, e4m3>(p, rows, stream) : by_size<f16, f16>(p, rows, stream);
  return cache_dtype == kE4M3 ? by_size<bf16, e4m3>(p, rows, stream) : by_size<bf16, bf16>(p, rows, stream);
}

}  // namespace samhip
