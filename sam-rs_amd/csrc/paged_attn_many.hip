// Paged attention on gfx950 for many rows a key head (a prompt's chunk, a frame's queries), f16 / bf16 queries over pages
// of their own type or of e4m3.
//
// Work: a workgroup of four waves takes 128 rows (new token x query head of one key head) and one range of keys; a wave
// owns 32 rows. Tiles of 64 keys go from their pages into LDS, the next one on its way while this one is worked on, two
// buffers each, one barrier a tile: 16-bit tiles that every row sees whole straight, others and e4m3 through registers
// (codes become 16-bit values with their row's scale on the way, once per workgroup). A lane looks one key of the tile up;
// the loads take their rows from that lane.
//   S^T = K Q^T on v_mfma_f32_32x32x16 with Q in registers: a lane holds one row's scores of 32 keys, so that softmax
//   needs one exchange between lane halves. O^T += V^T P^T takes the scores' registers as its B operand under a fixed
//   permutation of keys that the transposing reads of V (ds_read_b64_tr_b16) follow.
//
// A value that is not finite must not reach the rows that do not see its key (0 * inf = NaN). Tiles that some row does
// not see whole are looked over as they are stored: such values go into LDS as 0, and the rows that see one add it
// afterwards.
//
// Softmax statistics and sums are f32; the running maximum moves only when a tile passes it by 4 (in log2), so that O is
// rarely rescaled. f16 P is rounded to f16 and summed as rounded, all of it times 2^11, which O / l cancels: P then ends
// below 2^15, and weights keep f16's 11 bits down to 2^-25 of the largest, so that thousands of keys far below one that
// dominates are not lost (each is off by 2^-36 of it at most). A maximum that moves later would leave less of f16's range:
// 8192 rows and keys, 4 heads of 256 in f16 on a card a tenth slower: 358 us with 8, 348 with 4, 368, 386 and 441 with 3, 2
// and 0; at 128 319, 323, 321, 323 and 333.
// bf16 P goes as hi + lo, whose range is f32's. The exponent of a weight is one instruction, score * scale - maximum * scale,
// of which the latter is rounded: harmless up to 2^20, where it is off by 1/16, but from 2^24 on P would pass f16's range. A
// tile with such scores is computed again with (score - maximum) * scale, an instruction more a score (that form alone took
// 390 us at head dim 64 where this takes 371, 8192 rows and keys of 16 heads in f16, and 310 against 303 at 128 with 8).
//
// What bounds it: products, softmax and LDS reads beside each other on too few waves (a loop of the products alone, fed
// from LDS, reaches 1.11 PFLOP/s at head dim 128). Vector and matrix units are busy 60% and 33% of the cycles at head dim 64,
// 43% and 40% at 128, together nearly the whole time, also where more of them run beside each other: fewer instructions
// count, not a closer order. At 256, with one wave a SIMD, they are 33% and 32%, and the rest is waiting. 8192 rows over
// 8192 keys, f16: head dim 64 374 us (16 heads, 0.73 PFLOP/s), 96 259 (8 heads, 0.80), 128 309 (8 heads, 0.89), 256 337 (4
// heads, 0.82); bf16 at 64 542 (0.51), at 128 383 (0.72), with 1.5 times the products; e4m3 at 128 321 (0.86), at 256 374 (0.74),
// where 8 codes a load instead of 16 took 377 and 417. On a card a tenth slower kAhead 2 took 319, 279 and 370 us at 128, 96 and
// 256, and 4 317, 271 and 345.
#include <type_traits>

#include "lds_dma.hpp"
#include "paged.hpp"

namespace samhip {

namespace {

constexpr float kFarScore = 1048576.f;  // 2^20: below it, what rounds in f32 stays below 1/16
constexpr float kSlack = 4.f;  // how far a tile may pass the running maximum, in log2

// LDS: rows of 128, 256 or 512 bytes without padding, as the DMA leaves them (a wave's instruction fills 1 KB). 16-byte
// chunk c of row r lies at c ^ swizzle(r), so that the 16 rows of which a K read takes one chunk each, and the 8 rows of
// which a V read takes 64 bytes each, fall on all 64 banks alike.
template <int DP> struct ManyGeom {
  static constexpr int KS = DP / 16, MBO = DP / 32;
  static constexpr int ROW = DP <= 64 ? 128 : DP <= 128 ? 256 : 512;  // bytes
  static constexpr int BUF = 64 * ROW, LDS = 4 * BUF + 16;            // K0, K1, V0, V1, and two flags
  static constexpr int CPR = ROW / 16, RPI = 64 / CPR, PT = 16 / RPI; // chunks a row, rows an instruction, instructions
  static __device__ int kswz(int r) { return ROW == 128 ? (r >> 1) & 7 : r & 15; }
  static __device__ int vswz(int r) { return ROW == 128 ? (r >> 1 & 1) << 2 : (r & 3) << 2; }
};

// Lane l's 16 bytes at its own p land at LDS byte address lds + 16 l (lds wave-uniform; idle lanes leave theirs alone).
__device__ __forceinline__ void dma16_from(const void* p, unsigned lds) {
  asm volatile("s_mov_b32 m0, %1\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(p), "s"(lds) : "memory", "m0");
}

template <typename T, typename C, int DP>
__global__ __launch_bounds__(256, DP > 128 ? 1 : DP > 64 ? 2 : 3) void paged_many_kernel(PagedParams p) {
  typedef ManyGeom<DP> G;
  typedef typename Vec<T>::x8 X8;
  constexpr bool kCoded = __is_same(C, e4m3), kSplitP = __is_same(T, bf16);
  constexpr float kLift = kSplitP ? 0.f : 15.f - kSlack;  // P is lifted by 2^kLift
  // LDS fragments in flight ahead of their products: bf16 at head dim 64 has fewer registers for them (8192 rows
  // and keys, 16 heads: 561 us against 568 with four, from e4m3 577 against 608)
  constexpr int kAhead = DP <= 64 && kSplitP ? 2 : 4;
  typedef __attribute__((address_space(3))) X8 lds_x8;
  typedef __attribute__((address_space(3))) u32x4 lds_u32x4;
  constexpr int KS = G::KS, MBO = G::MBO, ROW = G::ROW, BUF = G::BUF, CPR = G::CPR, RPI = G::RPI, PT = G::PT;
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
  const unsigned lds0 = lds_addr(smem);
  int* odd = reinterpret_cast<int*>(smem + 4 * BUF);  // the tile in each buffer that went there without such values

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 31, hh = lane >> 5, g = lane >> 4, gi = lane & 15;
  const int d = p.c.d;
  if (p.zero_rest) paged_zero_rest<T>(p);
  const PagedWork w = paged_work(p);
  const int rows = w.lq * p.group;
  const C* kp = reinterpret_cast<const C*>(p.c.k);
  const C* vp = reinterpret_cast<const C*>(p.c.v);
  // Staging: instruction u of a wave moves rows srow(u) .. + RPI of a tile, lane l the chunk at position l % CPR of its row
  const int spos = lane % CPR;
  auto srow = [&](int u) { return 16 * wave + RPI * u + lane / CPR; };
  auto kcol = [&](int u) { return 8 * (spos ^ G::kswz(RPI * u + lane / CPR)); };
  auto vcol = [&](int u) { return 8 * (spos ^ G::vswz(RPI * u + lane / CPR)); };
  // e4m3: a load brings two chunks of a row, 16 codes, to the lane of LPR that stores them
  constexpr int CH = kCoded ? 2 : 1, PR = PT / CH, LPR = CPR / CH;
  const int rlane = lane / LPR, rcol = 8 * CH * (lane % LPR);
  auto rrow = [&](int u) { return 16 * wave + CH * RPI * u + rlane; };

  if (d < ROW / 2) {  // columns past d are never written: K's meet zeros of q, and V's only feed columns that are dropped
    for (int c = tid; c < 4 * BUF / 16; c += 256) *(lds_u32x4*)(size_t)(lds0 + 16 * c) = u32x4{};
  }

  for (int rt = w.tile; (long)rt * 128 < rows; rt += p.rtiles) {
    auto keys_of = [&](int r) {  // keys that row r sees
      const int t = (int)divide_magic(r, p.gmagic, p.gshift);
      return paged_keys(w, p.causal, t);
    };
    const int most = keys_of(min((rt + 1) * 128, rows) - 1);
    const int least = keys_of(rt * 128);
    const int wfirst = rt * 128 + 32 * wave;
    const bool rows_here = wfirst < rows;
    const int wleast = rows_here ? keys_of(wfirst) : 0, wmost = rows_here ? keys_of(min(wfirst + 32, rows) - 1) : 0;
    // blocks of 32 keys, as the other kernels count them; a tile is two
    const int tiles = (most + 63) >> 6, per = paged_share(tiles, (p.per + 1) >> 1, p.nsplit);
    const int t0 = min(tiles, w.split * per), t1 = min(tiles, t0 + per);
    const bool direct = tiles <= per;  // one split has all keys: it writes the result itself
    if (direct && w.split > 0) continue;

    // The tile's rows over this split's keys; false: its scores are too large for the short form of the exponent, and nothing
    // is written
    auto run = [&](auto far_scores) {
      constexpr bool kFar = decltype(far_scores)::value;
      const int r = min(wfirst + n, rows - 1);
      const int tk = (int)divide_magic(r, p.gmagic, p.gshift);
      const int limit = keys_of(r);
      const T* qr = reinterpret_cast<const T*>(p.q) + (w.s0 + tk) * p.sq[0] + (w.head * p.group + r - tk * p.group) * p.sq[1];

      // lane l's own key of a tile; a key that is not there reads row 0 and is masked (K) or cleared (V)
      auto entry_of = [&](int t) { return paged_entry(p.c, w.b, 64 * min(t, t1 - 1) + lane, most); };
      auto held = [&](int row) { return __builtin_amdgcn_ballot_w64(row >= 0); };
      auto whole = [&](int t, unsigned long there) { return 64 * t + 64 <= least && there == ~0ul; };
      // A tile that every row sees whole goes from its pages straight to LDS; one to be looked over, and e4m3, through
      // registers
      auto direct_to_lds = [&](int t, unsigned long there) { return !kCoded && whole(t, there); };
      auto dma = [&](int own, int buf) {
        unsigned row[PT];  // all there: the products below are one instruction each
  #pragma unroll
        for (int u = 0; u < PT; ++u) row[u] = (unsigned)__shfl(own, srow(u));
        auto rows_to = [&](const C* base, unsigned to, auto col) {
          if (d == ROW / 2) {
  #pragma unroll
            for (int u = 0; u < PT; ++u) dma16_from(base + (unsigned long)row[u] * (ROW / 2) + col(u), to + 1024 * u);
          } else {
  #pragma unroll
            for (int u = 0; u < PT; ++u)
              if (col(u) < d) dma16_from(base + (unsigned long)row[u] * (unsigned)d + col(u), to + 1024 * u);
          }
        };
        rows_to(kp, lds0 + buf * BUF + 16 * wave * ROW, kcol);
        rows_to(vp, lds0 + (2 + buf) * BUF + 16 * wave * ROW, vcol);
      };
      // e4m3: the next tile's chunks on their way beside this one's products. Else a tile that is looked over comes after
      // them, V once K is stored, in registers that the products have had.
      u32x4 kreg[PR], vbuf[kCoded ? PR : 1];
      u32x4* vreg = kCoded ? vbuf : kreg;
      unsigned char kscale = 127, vscale = 127;  // of the lane's own key
      auto load = [&](const C* base, const unsigned char* scales, int own, auto col, u32x4* reg, unsigned char& scale) {
        auto at = [&](int u) { return base + (unsigned long)(unsigned)max(__shfl(own, rrow(u)), 0) * (unsigned)d; };
        if constexpr (kCoded) {
          scale = scales[max(own, 0)];
          if (d % 16 == 0) {
  #pragma unroll
            for (int u = 0; u < PR; ++u) reg[u] = *reinterpret_cast<const u32x4*>(at(u) + min(rcol, d - 16));
          } else {  // a row's last chunk alone: 16 bytes would leave the row
  #pragma unroll
            for (int u = 0; u < PR; ++u) {
              const C* r = at(u);
              const u32x2 lo = *reinterpret_cast<const u32x2*>(r + min(rcol, d - 8)),
                          hi = *reinterpret_cast<const u32x2*>(r + min(rcol + 8, d - 8));
              reg[u] = u32x4{lo[0], lo[1], hi[0], hi[1]};
            }
          }
        } else {
  #pragma unroll
          for (int u = 0; u < PR; ++u) reg[u] = *reinterpret_cast<const u32x4*>(at(u) + min(col(u), d - 8));
        }
      };
      auto load_k = [&](int own) { load(kp, p.c.ks, own, kcol, kreg, kscale); };
      auto load_v = [&](int own) { load(vp, p.c.vs, own, vcol, vreg, vscale); };
      auto values = [&](const u32x4* reg, unsigned char scale, u32x4* x) {  // x[CH u + c]: chunk c of load u
        if constexpr (kCoded) {
          float f[PR];
          const float mine = pow2_of(scale);
  #pragma unroll
          for (int u = 0; u < PR; ++u) f[u] = __shfl(mine, rrow(u));  // all before their use: each takes LDS's latency
  #pragma unroll
          for (int u = 0; u < PR; ++u)
  #pragma unroll
            for (int c = 0; c < CH; ++c)
              x[CH * u + c] = u32x4{decode2<T, false>(reg[u][2 * c], f[u]), decode2<T, true>(reg[u][2 * c], f[u]),
                                    decode2<T, false>(reg[u][2 * c + 1], f[u]), decode2<T, true>(reg[u][2 * c + 1], f[u])};
        } else {
  #pragma unroll
          for (int u = 0; u < PR; ++u) x[u] = reg[u];
        }
      };
      // Chunk c of load u is for column col(u, c) and goes to its swizzled place: where the lane's own is, or, of e4m3, the
      // even chunk's place of the lane's first row with c and the row's part of the swizzle exclusive-ored in.
      auto chunk_col = [&](int u, int c, auto col) { return kCoded ? rcol + 8 * c : col(u); };
      auto store = [&](unsigned to, int u, int c, auto col, int lane_swz, int u_swz, u32x4 x) {
        const unsigned at = kCoded ? ((to + (16 * wave + rlane) * ROW + 16 * ((rcol / 8) ^ lane_swz)) ^ 16 * (c ^ u_swz)) + CH * RPI * ROW * u
                                   : to + 16 * wave * ROW + 16 * lane + 1024 * u;
        if (chunk_col(u, c, col) < d) *(lds_u32x4*)(size_t)at = x;
      };
      auto store_k = [&](int buf) {
        u32x4 x[PT];
        values(kreg, kscale, x);
  #pragma unroll
        for (int u = 0; u < PR; ++u)
  #pragma unroll
          for (int c = 0; c < CH; ++c) store(lds0 + buf * BUF, u, c, kcol, G::kswz(rlane), G::kswz(CH * RPI * u), x[CH * u + c]);
      };
      auto store_v = [&](int t, unsigned long there, int buf) {
        u32x4 x[PT];
        values(vreg, vscale, x);
        if (!whole(t, there)) {
          unsigned any = 0;
  #pragma unroll
          for (int u = 0; u < PR; ++u)
  #pragma unroll
            for (int c = 0; c < CH; ++c) {
              const bool ok = (there >> rrow(u) & 1) && chunk_col(u, c, vcol) < d;
  #pragma unroll
              for (int i = 0; i < 4; ++i) {
                const unsigned bad = not_finite2<T>(x[CH * u + c][i]);
                x[CH * u + c][i] = ok ? without2(x[CH * u + c][i], bad) : 0u;
                any |= ok ? bad : 0u;
              }
            }
          if (any) odd[buf] = t;
        }
  #pragma unroll
        for (int u = 0; u < PR; ++u)
  #pragma unroll
          for (int c = 0; c < CH; ++c) store(lds0 + (2 + buf) * BUF, u, c, vcol, G::vswz(rlane), G::vswz(CH * RPI * u), x[CH * u + c]);
      };

      // Table entries two tiles ahead, K and V one
      PagedEntry entry = {-1, -1};
      int own = -1;
      if (tid < 3) odd[tid] = tid < 2 ? -1 : 0;
      if (t0 < t1) {
        const PagedEntry first = entry_of(t0);
        entry = entry_of(t0 + 1);
        own = paged_row(p.c, first, w.head);
        load_k(own);
        if (kCoded) load_v(own);
      }
      X8 qf[KS];
  #pragma unroll
      for (int s = 0; s < KS; ++s) {
        const int c = 16 * s + 8 * hh;
        qf[s] = c < d ? *reinterpret_cast<const X8*>(qr + c) : X8{};
      }
      unsigned long there = held(own);
      __syncthreads();
      if (t0 < t1) {
        store_k(0);
        if (!kCoded) load_v(own);
        store_v(t0, there, 0);
      }
      // Q is here: told to the compiler, whose own wait for it would stand in the loop, behind the next tile's loads
      __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
      __syncthreads();

      // K (A operand of S^T): row 32 h + n, chunk 2 k + hh; the swizzle of the even part is an exclusive or with 32 k
      const unsigned kad = lds0 + n * ROW + 16 * (hh ^ G::kswz(n));
      // V^T (A operand of O^T): the transposing reads start at key 4 (g >> 1) + gi / 4, column 16 (g & 1) + 4 (gi & 3)
      const int vkey = 4 * (g >> 1) + (gi >> 2);
      const unsigned vad = lds0 + 2 * BUF + vkey * ROW + 16 * G::vswz(vkey) + 32 * (g & 1) + 8 * (gi & 3);
      const float sc = p.sc;
      float m = -INFINITY, l = 0.f, far = 0.f;
      f32x16 o[MBO];
  #pragma unroll
      for (int ob = 0; ob < MBO; ++ob) o[ob] = f32x16{};

      for (int t = t0; t < t1; ++t) {
        const int buf = (t - t0) & 1, key0 = 64 * t;
        const int next = paged_row(p.c, entry, w.head);
        const unsigned long coming = held(next);
        const bool more = t + 1 < t1, straight = direct_to_lds(t + 1, coming);
        entry = entry_of(t + 2);
        if (more) {
          if (straight) {
            dma(next, buf ^ 1);
          } else if (kCoded) {
            load_k(next);
            load_v(next);
          }
        }
        if (key0 < wmost) {
          const unsigned kb = kad + buf * BUF, vb = vad + buf * BUF;
          const bool masks = key0 + 64 > wleast || there != ~0ul;
          // The tile's two halves of 32 keys, one's softmax on the vector unit beside the other's products on the matrix
          // unit: S0 | S1 with softmax 0 | P0 V0 with softmax 1 | P1 V1. LDS fragments are read kAhead products before
          // their use. The scheduling groups hold these orders, which the compiler does not find. It moves a half's exponentials
          // behind the branch that may rescale O, to other waves' products: held before it they cost 3 to 6%.
          f32x16 s[2];
          X8 kf[2 * KS], vf[4 * MBO], b[4], blo[4];
          float alpha = 1.f;
          auto kread = [&](int i) { kf[i] = *(const lds_x8*)(size_t)((kb ^ 32 * (i % KS & 7)) + 256 * (i % KS >> 3) + 32 * ROW * (i / KS)); };
          auto vread = [&](int i) {  // keys 16 u + 8 (j / 4) + 4 hh + j % 4 of columns 32 ob ..; i = u MBO + ob
            const unsigned a = (vb ^ 64 * (i % MBO & 3)) + 256 * (i % MBO >> 2) + 16 * ROW * (i / MBO);
            vf[i] = join8<T>(lds_read_tr16_at(a), lds_read_tr16_at(a + 8 * ROW));
          };
          auto qk = [&](int i) {
            s[i / KS] = mma32(kf[i], qf[i % KS], i % KS == 0 ? f32x16{} : s[i / KS]);
            if (i + kAhead < 2 * KS) kread(i + kAhead);
          };
          auto pv = [&](int i) {
            o[i % MBO] = mma32(vf[i], b[i / MBO], o[i % MBO]);
            if constexpr (kSplitP) o[i % MBO] = mma32(vf[i], blo[i / MBO], o[i % MBO]);
            if (i + kAhead < 4 * MBO) vread(i + kAhead);
          };
          auto mask = [&](int h) {
            // shifted by the lane's part of the key, so that constants are left (the compiler would keep one key and one
            // bit a score in registers)
            const int lim = limit - key0 - 32 * h - 4 * hh;
            const unsigned bits = (unsigned)(there >> (32 * h)) >> (4 * hh);
  #pragma unroll
            for (int e = 0; e < 16; ++e) {
              const int kk = 8 * (e >> 2) + (e & 3);
              s[h][e] = kk < lim && (bits >> kk & 1) ? s[h][e] : -INFINITY;
            }
          };
          auto softmax = [&](int h) {  // of half h: b[2 h], b[2 h + 1], and alpha, by which O is to be scaled first
            float top = s[h][0];
  #pragma unroll
            for (int e = 1; e < 16; ++e) top = max_nc(top, s[h][e]);
            top = max_with_partner32(top);
            if constexpr (!kFar) top = top * sc - kLift;
            const float up = kFar ? (top - m) * sc : top - m, mn = up > kSlack ? top : m;
            const float base = mn == -INFINITY ? 0.f : mn;
            alpha = exp2_fast(kFar ? (m - base) * sc : m - base);  // m == mn: 1, or 0 while both are -inf and O is 0
            if constexpr (!kFar) far = fmaxf(far, fabsf(base));
            m = mn;
            l *= alpha;
  #pragma unroll
            for (int u = 2 * h; u < 2 * h + 2; ++u) {
              float pr[8];
  #pragma unroll
              for (int j = 0; j < 8; ++j) {
                const float x = s[h][8 * (u & 1) + j];
                pr[j] = exp2_fast(kFar ? fmaf(x - base, sc, kLift) : fmaf(x, sc, -base));
              }
              if constexpr (kSplitP) {
  #pragma unroll
                for (int j = 0; j < 8; ++j) l += pr[j];
                split_hi_lo(pr, b[u], blo[u]);
              } else {
                b[u] = pack8(pr, (X8*)nullptr);
                typedef _Float16 h2 __attribute__((ext_vector_type(2)));
  #pragma unroll
                for (int j = 0; j < 8; j += 2)
                  l = __builtin_amdgcn_fdot2(h2{b[u][j], b[u][j + 1]}, h2{(f16)1.f, (f16)1.f}, l, false);
              }
            }
          };
          auto rescale = [&]() {
            if (wave_any(alpha != 1.f)) {
  #pragma unroll
              for (int ob = 0; ob < MBO; ++ob) o[ob] *= alpha;
            }
          };
          constexpr int kVec = (kSplitP ? 96 : 48), kTrans = 17;  // a half's softmax, in vector and exponential instructions
          __builtin_amdgcn_sched_barrier(0);
  #pragma unroll
          for (int i = 0; i < kAhead; ++i) kread(i);
  #pragma unroll
          for (int i = 0; i < KS; ++i) qk(i);
          __builtin_amdgcn_sched_group_barrier(0x100, kAhead, 0);
  #pragma unroll
          for (int i = 0; i < KS; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
          }
          __builtin_amdgcn_sched_barrier(0);
          if (masks) mask(0);
          __builtin_amdgcn_sched_barrier(0);
          softmax(0);
  #pragma unroll
          for (int i = KS; i < 2 * KS; ++i) qk(i);
  #pragma unroll
          for (int i = 0; i < kAhead; ++i) vread(i);
  #pragma unroll
          for (int i = KS; i < 2 * KS; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x002, (kVec + KS - 1) / KS, 0);
            __builtin_amdgcn_sched_group_barrier(0x400, (kTrans + KS - 1) / KS, 0);
          }
          __builtin_amdgcn_sched_barrier(0);
          rescale();
          if (masks) mask(1);
          __builtin_amdgcn_sched_barrier(0);
          softmax(1);
  #pragma unroll
          for (int i = 0; i < 2 * MBO; ++i) pv(i);
  #pragma unroll
          for (int i = 0; i < 2 * MBO; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x008, kSplitP ? 2 : 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
            __builtin_amdgcn_sched_group_barrier(0x002, (kVec + 2 * MBO - 1) / (2 * MBO), 0);
            __builtin_amdgcn_sched_group_barrier(0x400, (kTrans + 2 * MBO - 1) / (2 * MBO), 0);
          }
          __builtin_amdgcn_sched_barrier(0);
          rescale();
          __builtin_amdgcn_sched_barrier(0);
  #pragma unroll
          for (int i = 2 * MBO; i < 4 * MBO; ++i) pv(i);
  #pragma unroll
          for (int i = 2 * MBO; i < 4 * MBO; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x008, kSplitP ? 2 : 1, 0);
            if (i + kAhead < 4 * MBO) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
          }
          __builtin_amdgcn_sched_barrier(0);
          if (!whole(t, there) && odd[buf] == t) {
            for (int kk = 0; kk < 64; ++kk) {
              if (!(there >> kk & 1)) continue;
              const int row = __shfl(own, kk);
              const float vs = kCoded ? pow2_of(p.c.vs[row]) : 1.f;
              const bool sees = key0 + kk < limit;
  #pragma unroll
              for (int ob = 0; ob < MBO; ++ob)
  #pragma unroll
                for (int a = 0; a < 4; ++a) {
                  const int col = 32 * ob + 8 * a + 4 * hh;
                  if (col < d) {
                    const f32x4 x = only_not_finite4<T>(vp + (long)row * d + col, vs);
  #pragma unroll
                    for (int e = 0; e < 4; ++e) o[ob][4 * a + e] += sees ? x[e] : 0.f;
                  }
                }
            }
          }
        }
        if (more && !straight) {
          if (!kCoded) load_k(next);
          store_k(buf ^ 1);
          if (!kCoded) load_v(next);
          store_v(t + 1, coming, buf ^ 1);
        }
        own = next;
        there = coming;
        if constexpr (!kFar) {
          if (!more && wave_any(far >= kFarScore)) odd[2] = 1;
        }
        wait_vm<0>();  // the tile on its way to LDS
        __syncthreads();
      }
      if constexpr (!kFar) {
        if (odd[2]) {
          __syncthreads();  // the second pass sets it back
          return false;
        }
      }

      // lane holds O^T[32 ob + 8 a + 4 hh + e][row n] in o[ob][4 a + e]
      l = sum_with_partner32(l);
      if (wfirst + n < rows) {
        const long tok = w.s0 + tk;
        const int hq = w.head * p.group + (r - tk * p.group);
        const float inv = l == 0.f ? 0.f : 1.f / l;  // a row that sees no key is 0
        const long part = (w.split * (long)p.tokens + tok) * p.heads + hq;
        auto columns = [&](auto put) {
  #pragma unroll
          for (int ob = 0; ob < MBO; ++ob)
  #pragma unroll
            for (int a = 0; a < 4; ++a)
              if (32 * ob + 8 * a + 4 * hh < d)
                put(32 * ob + 8 * a + 4 * hh, f32x4{o[ob][4 * a], o[ob][4 * a + 1], o[ob][4 * a + 2], o[ob][4 * a + 3]});
        };
        if (direct) {
          T* to = reinterpret_cast<T*>(p.out) + tok * p.so[0] + hq * p.so[1];
          columns([&](int col, f32x4 x) {
            typename Vec<T>::x4 y;
  #pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = from_f32<T>(f32_result(x[e] * inv));
            *reinterpret_cast<typename Vec<T>::x4*>(to + col) = y;
          });
        } else if (t0 < t1) {
          columns([&](int col, f32x4 x) { *reinterpret_cast<f32x4*>(p.opart + part * d + col) = x; });
        }
        if (p.nsplit > 1 && hh == 0) *reinterpret_cast<float2*>(p.ml + 2 * part) = direct ? float2{0.f, -1.f} : float2{kFar ? m * sc - kLift : m, l};
      }
      __syncthreads();  // the next rows' first tile replaces buffer 0
      return true;
    };
    if (!run(std::false_type{})) run(std::true_type{});
  }
}

template <typename T, typename C, int DP> hipError_t launch_many(const PagedParams& p, hipStream_t stream) {
  auto kern = paged_many_kernel<T, C, DP>;
  static std::atomic<unsigned long long> done;  // opt-in to more than 64 KB of dynamic LDS
  if (const hipError_t e = lds_opt_in(done, (const void*)kern, ManyGeom<DP>::LDS); e != hipSuccess) return e;
  const long blocks = (long)p.rtiles * p.nsplit * p.c.heads * p.c.batch;
  hipLaunchKernelGGL(kern, dim3((unsigned)blocks), dim3(256), ManyGeom<DP>::LDS, stream, p);
  return hipGetLastError();
}
template <typename T, typename C> hipError_t by_size(const PagedParams& p, hipStream_t stream) {
  const int d = p.c.d;
  return d <= 64 ? launch_many<T, C, 64>(p, stream)
                 : d <= 96 ? launch_many<T, C, 96>(p, stream)
                           : d <= 128 ? launch_many<T, C, 128>(p, stream) : launch_many<T, C, 256>(p, stream);
}

}  // namespace

hipError_t paged_many(int dtype, int cache_dtype, const PagedParams& p, hipStream_t stream) {
  if (dtype == kF16)
    return cache_dtype == kE4M3 ? by_size<f16, e4m3>(p, stream) : by_size<f16, f16>(p, stream);
  return cache_dtype == kE4M3 ? by_size<bf16, e4m3>(p, stream) : by_size<bf16, bf16>(p, stream);
}

}  // namespace samhip
