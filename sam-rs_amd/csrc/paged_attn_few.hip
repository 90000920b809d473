// Paged attention on gfx950 for few rows a key head (a decoding step, a short chunk), f16 / bf16 queries over pages of
// their own type, of e4m3 or of e2m1.
//
// What bounds it: the bytes of K and V, each used for 4 flops a row. So nothing stands between memory and the matrix
// units: a wave takes blocks of 32 keys of its workgroup's range, loads their K and V rows straight into registers, the
// next block's K while it weighs this one's V and the next V during the next scores, and passes neither through LDS.
//   S^T = K Q^T on v_mfma_f32_16x16x32: a lane's 16 bytes (8 codes) of key row n are an A operand as they are.
//   O^T += V^T P^T: a lane loads the same few columns of 8 keys, whose 16-bit pairs v_perm_b32 transposes in registers
//   into A operands (the output's columns come out permuted, which the store undoes); P stays where S^T left it, since
//   the reduction index is permuted alike: element j of lane group g is key 16 (j / 4) + 4 g + j % 4.
// e4m3 codes become 16-bit values with their row's scale in one conversion, exactly (in f16, values below 2^-14 to
// f16's subnormal step), and so do e2m1's with their block's. Softmax statistics and sums are f32. f16 P is rounded to f16 and
// its sum taken over the rounded values: results of N(0, 1) keys and values are off by 2.5e-4 to 2.8e-4 of their size, of which their
// own rounding is 2.1e-4, and a second term would double the products of V, as bf16's does. All of it is taken times 2^15, which O / l cancels: weights keep f16's 11 bits down to 2^-29 of the largest, so that
// thousands of keys far below one that dominates are not lost (each is off by 2^-40 of it at most). The exponent is taken of
// (score - maximum) * scale, so that scores of any size keep P in f16's range. bf16 P goes as
// hi + lo, which leaves 2^-16 of it (one bf16 term would leave 2^-8, as much as the output's own rounding).
//
// The four waves of a workgroup join at its end, the key ranges of a sequence in paged_combine_kernel.
//
// Measured, 32 sequences of 8192 keys, 8 key heads of 128, one token of 4 query heads a key head: f16 pages 187 us (5.7
// TB/s), e4m3 pages 107 with f16 queries and 123 with bf16 (5.0 and 4.4; not for their instructions: a fifth fewer took as
// long). 64-key blocks of e4m3 were no faster. e2m1 pages 55 us with f16 queries and 66 with bf16 (5.2 and 4.3 TB/s): half of
// the bytes of e4m3, so that instructions (conversions, transposition, the exponentials, bf16's two products) bound it as
// much as memory does; a wave of head dim 64 takes two blocks at a time, whose latencies overlap.
#include <type_traits>

#include "lds_dma.hpp"
#include "paged.hpp"

namespace samhip {

namespace {

template <int BYTES> struct Raw;
template <> struct Raw<2> {
  typedef unsigned short t;
};
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
constexpr int few_workgroups(bool wide, int dp, int rb) { return dp * rb > 128 ? 1 : dp == 128 && wide ? 2 : 3; }

// QUADS (e2m1 of a full head dim, pages of whole quads): the four neighbouring keys of a lane follow one another in their
// page, so that a quad has one address, its rows lie at constant offsets and their scales are one load.
template <typename T, typename C, int DP, int RB, bool QUADS>
__global__ __launch_bounds__(256, few_workgroups(sizeof(C) > 1, DP, RB)) void paged_few_kernel(PagedParams p) {
  typedef typename Vec<T>::x8 X8;
  constexpr bool kMx = __is_same(C, e2m1), kCoded = __is_same(C, e4m3), kSplitP = __is_same(T, bf16);
  constexpr float kLift = kSplitP ? 0.f : 15.f;  // P is lifted by 2^kLift
  constexpr int TR = 16 * RB, NK = DP / 32;
  constexpr int CW = DP >= 128 ? 8 : DP / 16, NV = DP / (16 * CW);  // columns of a value row that a lane takes at once
  typedef typename Raw<held_bytes<C>(8)>::t KRaw;
  typedef typename Raw<held_bytes<C>(CW)>::t VRaw;
  // e2m1: a lane's words of a key row lie side by side, DP / 4 columns, so that they are one load or two and have one scale
  // or two; q's columns follow
  constexpr int KL = NK < 4 ? NK : 4, KSC = DP <= 128 ? 1 : 2;  // words of a load, scales of a lane
  constexpr int VSC = DP / 64;                                  // scales of a value row that a lane fetches
  constexpr int KB = QUADS && DP * RB == 64 ? 2 : 1, KEYS = 32 * KB;  // blocks and keys of an iteration
  typedef typename std::conditional<KB == 2, unsigned long, unsigned>::type Bits;  // one of each key
  __shared__ float sm_m[2][TR], sm_l[2][TR];
  __shared__ __attribute__((aligned(16))) float sm_o[2][RB * DP / 16][256];
  // bf16 over e2m1 at head dim 128 reads its queries from LDS for each block: in registers they leave room for two workgroups a
  // CU, not three (32 sequences of 820 to 8192 keys 55 and 51 us; f16, with three either way, 46 and 47)
  constexpr bool kQInLds = kMx && kSplitP && DP == 128 && RB == 1;
  __shared__ __attribute__((aligned(16))) u32x4 sm_q[kQInLds ? NK : 1][64];
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
    X8 qf[RB][kQInLds ? 1 : NK];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      const int r = min(rt * TR + 16 * rb + n, rows - 1);
      const int t = (int)divide_magic(r, p.gmagic, p.gshift);
      limit[rb] = paged_keys(w, p.causal, t);
      const T* qr = reinterpret_cast<const T*>(p.q) + (w.s0 + t) * p.sq[0] + (w.head * p.group + r - t * p.group) * p.sq[1];
#pragma unroll
      for (int c = 0; c < NK; ++c) {
        const int col = kMx ? DP / 4 * g + 8 * c : 32 * c + 8 * g;
        const X8 x = col < d ? *reinterpret_cast<const X8*>(qr + col) : X8{};
        if constexpr (kQInLds) {
          if (wave == 0) sm_q[c][lane] = __builtin_bit_cast(u32x4, x);
        } else {
          qf[rb][c] = x;
        }
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
    auto entry_of = [&](int blk) {
      return paged_entry(p.c, w.b, 32 * min(KB == 2 ? blk + (lane >> 5) : blk, b1 - 1) + (lane & 31), most);
    };
    auto row_of = [&](const PagedEntry& e, int blk) {
      const int r = paged_row(p.c, e, w.head);
      return KB == 2 && blk + (lane >> 5) >= b1 ? -1 : r;  // the range may end between two blocks
    };
    KRaw kx[2 * KB][NK];
    VRaw vx[8 * KB][NV];
    unsigned char ksx = 127, vsx = 127;  // scales of the lane's own key
    // e2m1: the scales of the lane's key blocks, and of half of its own key's value blocks (lanes 0 .. 31 the lower half of
    // each 128 columns' four, or of two)
    unsigned char kmx[2 * KB][KSC], vmx[VSC];
    // QUADS: of the lane's four neighbouring value rows, all of them: a row's DP / 32 bytes one after the other
    u32x2 vq[2 * KB][QUADS ? VSC : 1];
    const int G = d / kMxBlock;
    auto load_k = [&](int row) {
      if constexpr (kMx) {
#pragma unroll
        for (int i = 0; i < 2 * KB; ++i) {
          const int r = max(from_n(i, row), 0);
          const unsigned char* kr = reinterpret_cast<const unsigned char*>(kp) + (unsigned long)(unsigned)r * (unsigned)(d / 2);
#pragma unroll
          for (int c = 0; c < NK; c += KL) {
            const int at = min(DP / 4 * g + 8 * c, d - 8 * KL) / 2;
            if constexpr (KL == 2)
              *reinterpret_cast<u32x2*>(&kx[i][c]) = *reinterpret_cast<const u32x2*>(kr + at);
            else
              *reinterpret_cast<u32x4*>(&kx[i][c]) = *reinterpret_cast<const u32x4*>(kr + at);
          }
#pragma unroll
          for (int b = 0; b < KSC; ++b)
            kmx[i][b] = p.c.ks[(unsigned long)(unsigned)r * (unsigned)G + (unsigned)min(DP / 4 * g / kMxBlock + b, G - 1)];
        }
        return;
      }
      if constexpr (kCoded) ksx = p.c.ks[max(row, 0)];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const C* kr = kp + (long)max(from_n(i, row), 0) * d;
#pragma unroll
        for (int c = 0; c < NK; ++c) kx[i][c] = *reinterpret_cast<const KRaw*>(kr + min(32 * c + 8 * g, d - 8));
      }
    };
    auto load_v = [&](int row) {
      if constexpr (QUADS) {
#pragma unroll
        for (int i = 0; i < 2 * KB; ++i) {
          const unsigned long r = (unsigned)max(from_key(4 * i, row), 0);  // its three neighbours follow it in its page
          const C* vr = vp + r * (DP / 2);
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int q = 0; q < NV; ++q) vx[4 * i + j][q] = *reinterpret_cast<const VRaw*>(vr + j * (DP / 2) + CW / 2 * (16 * q + n));
          const u32x2* vs = reinterpret_cast<const u32x2*>(p.c.vs + r * (DP / kMxBlock));
#pragma unroll
          for (int b = 0; b < VSC; ++b) vq[i][b] = vs[b];
        }
        return;
      }
      if constexpr (kMx) {
        const unsigned char* vs = p.c.vs + (unsigned long)(unsigned)max(row, 0) * (unsigned)G;
#pragma unroll
        for (int b = 0; b < VSC; ++b) vmx[b] = vs[min(DP == 64 ? lane >> 5 : 4 * (b >> 1) + 2 * (lane >> 5) + (b & 1), G - 1)];
      }
      if constexpr (kCoded) vsx = p.c.vs[max(row, 0)];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const C* vr = held_at(vp, (long)max(from_key(j, row), 0) * d);
#pragma unroll
        for (int q = 0; q < NV; ++q) vx[j][q] = *reinterpret_cast<const VRaw*>(held_at(vr, min(CW * (16 * q + n), d - CW)));
      }
    };

    // Table entries two blocks ahead, K and V one: a wait for a load waits for those before it too, so the entries go
    // ahead of the rows that they are not needed for. After its last block a wave loads the range's last again: loads under
    // a condition would have the next scores wait for V too, as the compiler counts what is in flight on the shorter path.
    int row = -1;
    PagedEntry coming = {-1, -1};
    if (b0 + KB * wave < b1) {
      const PagedEntry first = entry_of(b0 + KB * wave);
      coming = entry_of(b0 + KB * (wave + 4));
      row = row_of(first, b0 + KB * wave);
      load_k(row);
      load_v(row);
    }
    // Q is here: told to the compiler, whose own wait for it would stand in the loop, behind the next block's loads
    __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
    if constexpr (kQInLds) __syncthreads();
    for (int blk = b0 + KB * wave; blk < b1; blk += 4 * KB) {
      const int key0 = 32 * blk;
      const int next = row_of(coming, blk + 4 * KB);
      coming = entry_of(blk + 8 * KB);
      const Bits there = (Bits)__builtin_amdgcn_ballot_w64(row >= 0);
      f32x4 s[RB][2 * KB];
      X8 ql[kQInLds ? NK : 1];
      if constexpr (kQInLds) {
        typedef __attribute__((address_space(3))) X8 lds_x8;
        const unsigned at = opaque(lds_addr(sm_q) + 16 * lane);  // hidden: not to be read once for all blocks
#pragma unroll
        for (int c = 0; c < NK; ++c) ql[c] = *(const lds_x8*)(size_t)(at + 1024 * c);
      }
      const float kso = kCoded ? pow2_of(ksx) : 1.f, vso = kCoded ? pow2_of(vsx) : 1.f;
      unsigned vmo = 0;
      if constexpr (kMx && !QUADS) {
#pragma unroll
        for (int b = 0; b < VSC; ++b) vmo |= (unsigned)vmx[b] << (8 * b);
      }
#pragma unroll
      for (int i = 0; i < 2 * KB; ++i) {
        float ks = 1.f;
        if constexpr (kCoded) ks = __int_as_float(from_n(i, __float_as_int(kso)));
#pragma unroll
        for (int c = 0; c < NK; ++c) {
          u32x4 a;
          if constexpr (kMx) {
            const float f = mx_scale(kmx[i][8 * c / kMxBlock % KSC]);
            a = u32x4{mx_decode2<T, 0>(kx[i][c], f), mx_decode2<T, 1>(kx[i][c], f), mx_decode2<T, 2>(kx[i][c], f), mx_decode2<T, 3>(kx[i][c], f)};
          } else if constexpr (kCoded)
            a = u32x4{decode2<T, false>(kx[i][c][0], ks), decode2<T, true>(kx[i][c][0], ks),
                      decode2<T, false>(kx[i][c][1], ks), decode2<T, true>(kx[i][c][1], ks)};
          else
            a = kx[i][c];
          if (kMx ? DP / 4 * g + 8 * c >= d : 32 * c + 32 > d && 32 * c + 8 * g >= d) a = u32x4{};
#pragma unroll
          for (int rb = 0; rb < RB; ++rb)
            s[rb][i] = mma16(__builtin_bit_cast(X8, a), kQInLds ? ql[kQInLds ? c : 0] : qf[rb][kQInLds ? 0 : c], c == 0 ? f32x4{} : s[rb][i]);
        }
      }
      // s[rb][i][e]: key key0 + 16 i + 4 g + e, row 16 rb + n
      load_k(next);  // in flight while this block's V is weighed
      const bool part = key0 + KEYS > least || there != (Bits)~(Bits)0;
      const Bits mine = there >> (4 * g);  // bit 16 i + e: the lane's key 16 i + 4 g + e
      X8 b[KB][RB], blo[KB][RB];
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) {
        float top = -INFINITY;
        if (part) {
#pragma unroll
          for (int i = 0; i < 2 * KB; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int kk = 16 * i + e;
              s[rb][i][e] = kk < limit[rb] - key0 - 4 * g && (mine >> kk & 1) ? s[rb][i][e] : -INFINITY;
            }
        }
#pragma unroll
        for (int i = 0; i < 2 * KB; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) top = max_nc(top, s[rb][i][e]);
        const float m_new = fmaxf(m[rb], max_over_rows16(top));
        const float base = m_new == -INFINITY ? 0.f : m_new;
        const float alpha = exp2_fast((m[rb] - base) * p.sc);
        m[rb] = m_new;
        l[rb] *= alpha;
        if (!kMx || wave_any(alpha != 1.f)) {
#pragma unroll
          for (int i = 0; i < DP / 16; ++i) o[rb][i] *= alpha;
        }
#pragma unroll
        for (int u = 0; u < KB; ++u) {
          float pv[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            pv[j] = exp2_fast(fmaf(s[rb][2 * u + (j >> 2)][j & 3] - base, p.sc, kLift));
          }
          if constexpr (kSplitP) {
#pragma unroll
            for (int j = 0; j < 8; ++j) l[rb] += pv[j];
            split_hi_lo(pv, b[u][rb], blo[u][rb]);
          } else {
            b[u][rb] = pack8(pv, (X8*)nullptr);
#pragma unroll
            for (int j = 0; j < 8; j += 2)
              l[rb] = __builtin_amdgcn_fdot2(f16x2{b[u][rb][j], b[u][rb][j + 1]}, f16x2{(f16)1.f, (f16)1.f}, l[rb], false);
          }
        }
      }
      unsigned odd = 0;
      float vs[8];
      if constexpr (kCoded) {
#pragma unroll
        for (int j = 0; j < 8; ++j) vs[j] = __int_as_float(from_key(j, __float_as_int(vso)));
      }
      unsigned vm[8];
      if constexpr (kMx && !QUADS) {  // the lane's blocks' half of the four
#pragma unroll
        for (int j = 0; j < 8; ++j) vm[j] = (unsigned)__builtin_amdgcn_ds_bpermute((int)at_g + 128 * (n >> 3) + 64 * (j >> 2) + 4 * (j & 3), (int)vmo);
      }
      if constexpr (kMx) {
        // columns 4 H .. 4 H + 3 of a lane's words: with all eight at a time, bf16 at head dim 128 spills at three
        // workgroups a CU
        auto columns = [&](auto half, int u, int q, const float* f) {
          constexpr int H = decltype(half)::value;
          unsigned v[8][2];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            v[j][0] = mx_decode2<T, 2 * H>(vx[8 * u + j][q], f[j]);
            v[j][1] = mx_decode2<T, 2 * H + 1>(vx[8 * u + j][q], f[j]);
          }
          if (part) {  // rows that are not there hold anything; values that are not finite go apart
            __builtin_amdgcn_sched_barrier(0);  // one branch, where the compiler would make one of each key's part
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const bool ok = mine >> (32 * u + 16 * (j >> 2) + (j & 3)) & 1;
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const unsigned bad = not_finite2<T>(v[j][h]);
                v[j][h] = ok ? without2(v[j][h], bad) : 0u;
                odd |= ok ? bad : 0u;
              }
            }
          }
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            u32x4 a;
#pragma unroll
            for (int j = 0; j < 4; ++j)  // keys 2 j and 2 j + 1 of column c
              a[j] = __builtin_amdgcn_perm(v[2 * j + 1][c >> 1], v[2 * j][c >> 1], c & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
              f32x4& acc = o[rb][q * CW + 4 * H + c];
              acc = mma16(__builtin_bit_cast(X8, a), b[u][rb], acc);
              if constexpr (kSplitP) acc = mma16(__builtin_bit_cast(X8, a), blo[u][rb], acc);
            }
          }
        };
#pragma unroll
        for (int uq = 0; uq < KB * NV; ++uq) {
          const int u = uq / NV, q = uq % NV;
          float f[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            if constexpr (QUADS) {
              const int at = (j & 3) * (DP / 64) + 2 * q;  // in pairs of the four rows' scales
              f[j] = mx_scale(__builtin_amdgcn_ubfe(vq[2 * u + (j >> 2)][at / 4][at / 2 % 2], DP == 64 ? 16 * (at & 1) + 8 * (n >> 3) : 8 * (n >> 2), 8));
            } else {
              f[j] = mx_scale(vm[j] >> (DP == 64 ? 0 : 16 * q + 8 * (n >> 2 & 1)) & 255);
            }
          }
          columns(std::integral_constant<int, 0>{}, u, q, f);
          if constexpr (CW == 8) {
            __builtin_amdgcn_sched_barrier(0);
            columns(std::integral_constant<int, 1>{}, u, q, f);
          }
        }
      } else {
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
              acc = mma16(__builtin_bit_cast(X8, a), b[0][rb], acc);
              if constexpr (kSplitP) acc = mma16(__builtin_bit_cast(X8, a), blo[0][rb], acc);
            }
          }
        }
      }
      if (wave_any(odd != 0)) {
        // A value that is not finite must not reach the rows that do not see its key (0 * inf = NaN): it was taken out
        // above, and the rows that see it add it here
        for (int kk = 0; kk < KEYS; ++kk) {
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
                  const float f = kMx ? mx_scale(p.c.vs[(unsigned long)(unsigned)kr * (unsigned)G + (unsigned)(col / kMxBlock)]) : s1;
                  const f32x4 x = only_not_finite4<T>(held_at(vp, (long)kr * d + col), f);
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
  auto run = [&](auto kern) { hipLaunchKernelGGL(kern, dim3((unsigned)blocks), dim3(256), 0, stream, p); };
  if (__is_same(C, e2m1) && p.c.d == DP && p.c.page % 4 == 0 && reinterpret_cast<uintptr_t>(p.c.vs) % 8 == 0)
    run(paged_few_kernel<T, C, DP, RB, __is_same(C, e2m1)>);
  else
    run(paged_few_kernel<T, C, DP, RB, false>);
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
  if (cache_dtype == kE2M1) return dtype == kF16 ? by_size<f16, e2m1>(p, rows, stream) : by_size<bf16, e2m1>(p, rows, stream);
  if (dtype == kF16)
    return cache_dtype == kE4M3 ? by_size<f16, e4m3>(p, rows, stream) : by_size<f16, f16>(p, rows, stream);
  return cache_dtype == kE4M3 ? by_size<bf16, e4m3>(p, rows, stream) : by_size<bf16, bf16>(p, rows, stream);
}

}  // namespace samhip
