// Paged attention on gfx950 for many rows a key head (a prompt's chunk, a frame's queries), f16 / bf16 queries over pages
// of their own type or of e4m3.
//
// Work: a workgroup of four waves takes 128 rows (new token x query head of one key head) and one range of keys; a wave
// owns 32 rows. Tiles of 64 keys go from their pages through registers into LDS, the next tile's loads in flight while
// this one is worked on (e4m3 codes become 16-bit values with their row's scale on the way, once per workgroup), two
// buffers each, one barrier a tile. A lane looks one key of the tile up; the loads take their rows from that lane.
//   S^T = K Q^T on v_mfma_f32_32x32x16 with Q in registers: a lane holds one row's scores of 32 keys, so that softmax
//   needs one exchange between lane halves. O^T += V^T P^T takes the scores' registers as its B operand under a fixed
//   permutation of keys that the transposing reads of V (ds_read_b64_tr_b16) follow.
//
// A value that is not finite must not reach the rows that do not see its key (0 * inf = NaN). Tiles that some row does
// not see whole are looked over as they are stored: such values go into LDS as 0, and the rows that see one add it
// afterwards.
//
// Softmax statistics and sums are f32; the running maximum moves only when a tile passes it by 8 (in log2), so that O is
// rarely rescaled. f16 P is rounded to f16 and summed as rounded; bf16 P goes as hi + lo.
#include <type_traits>

#include "lds_dma.hpp"
#include "paged.hpp"

namespace samhip {

namespace {

constexpr float kSlack = 8.f;
constexpr int kAhead = 4;  // LDS fragments in flight ahead of their products

template <int DP> struct ManyGeom {
  static constexpr int KS = DP / 16, MBO = DP / 32;
  static constexpr int KSTR = DP + 8;                     // K row stride (elements): rows 16 bytes apart mod 128
  static constexpr int VSTR = DP + (MBO == 3 ? 0 : 32);   // 16 or 48 banks mod 64 for the transposing reads
  static constexpr int KBUF = 64 * KSTR, VBUF = 64 * VSTR;
  static constexpr int LDS = 2 * (KBUF + VBUF) * 2;
  static constexpr int CPR = DP <= 64 ? 8 : DP <= 128 ? 16 : 32;  // threads to a row, 8 columns each
  static constexpr int RS = 256 / CPR, PT = 64 / RS;      // rows a round, rounds a tile
};

template <typename T, typename C, int DP>
__global__ __launch_bounds__(256, DP > 128 ? 1 : 2) void paged_many_kernel(PagedParams p) {
  typedef ManyGeom<DP> G;
  typedef typename Vec<T>::x8 X8;
  constexpr bool kCoded = __is_same(C, e4m3), kSplitP = __is_same(T, bf16);
  constexpr int KS = G::KS, MBO = G::MBO, KSTR = G::KSTR, VSTR = G::VSTR, CPR = G::CPR, RS = G::RS, PT = G::PT;
  __shared__ int odd[2];  // the tile in each buffer that was stored without values that are not finite
  typedef typename std::conditional<kCoded, u32x2, u32x4>::type Raw;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  T* ks_base = reinterpret_cast<T*>(smem);
  T* vs_base = ks_base + 2 * G::KBUF;

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 31, hh = lane >> 5, g = lane >> 4, gi = lane & 15;
  const int d = p.c.d;
  if (p.zero_rest) paged_zero_rest<T>(p);
  const PagedWork w = paged_work(p);
  const int rows = w.lq * p.group;
  const C* kp = reinterpret_cast<const C*>(p.c.k);
  const C* vp = reinterpret_cast<const C*>(p.c.v);
  const int srow = tid / CPR, scol = tid % CPR * 8;  // this thread's first row of a tile, and its columns
  const bool sin = scol < d;

  if (d < DP) {  // K's columns past d meet zeros of q, so they must be finite; V's only feed columns that are dropped
    for (int c = tid; c < 2 * 64 * (DP / 8); c += 256) {
      const int r = c / (DP / 8), c8 = c % (DP / 8) * 8;
      if (c8 >= d) *reinterpret_cast<u32x4*>(ks_base + (r >> 6) * G::KBUF + (r & 63) * KSTR + c8) = u32x4{};
    }
  }

  for (int rt = w.tile; (long)rt * 128 < rows; rt += p.rtiles) {
    auto keys_of = [&](int r) {  // keys that row r sees
      const int t = (int)divide_magic(r, p.gmagic, p.gshift);
      return p.causal ? max(0, min(w.len, w.len - w.lq + t + 1)) : w.len;
    };
    const int most = keys_of(min((rt + 1) * 128, rows) - 1);
    const int least = keys_of(rt * 128);
    const int wfirst = rt * 128 + 32 * wave;
    const bool rows_here = wfirst < rows;
    const int wleast = rows_here ? keys_of(wfirst) : 0, wmost = rows_here ? keys_of(min(wfirst + 32, rows) - 1) : 0;
    // blocks of 32 keys, as the other kernels count them; a tile is two
    const int tiles = (most + 63) >> 6, per = max((p.per + 1) >> 1, (tiles + p.nsplit - 1) / p.nsplit);
    const int t0 = min(tiles, w.split * per), t1 = min(tiles, t0 + per);
    const bool direct = tiles <= per;  // one split has all keys: it writes the result itself
    if (direct && w.split > 0) continue;

    const int r = min(wfirst + n, rows - 1);
    const int tk = (int)divide_magic(r, p.gmagic, p.gshift);
    const int limit = keys_of(r);
    const T* qr = reinterpret_cast<const T*>(p.q) + (w.s0 + tk) * p.sq[0] + (w.head * p.group + r - tk * p.group) * p.sq[1];

    // the next tile's chunks on their way, and in 8 bits the scales of the lane's own key
    struct Chunks {
      Raw x[PT];
      unsigned char scale;
    } kreg, vreg;
    // lane l's own key of a tile; a key that is not there reads row 0 and is masked (K) or cleared (V)
    auto entry_of = [&](int t) { return paged_entry(p.c, w.b, 64 * min(t, t1 - 1) + lane, most); };
    auto load = [&](int own) {
      if constexpr (kCoded) {
        kreg.scale = p.c.ks[max(own, 0)];
        vreg.scale = p.c.vs[max(own, 0)];
      }
      long off[PT];
#pragma unroll
      for (int u = 0; u < PT; ++u) off[u] = (long)max(__shfl(own, srow + u * RS), 0) * d + min(scol, d - 8);
#pragma unroll
      for (int u = 0; u < PT; ++u) kreg.x[u] = *reinterpret_cast<const Raw*>(kp + off[u]);
#pragma unroll
      for (int u = 0; u < PT; ++u) vreg.x[u] = *reinterpret_cast<const Raw*>(vp + off[u]);
    };
    auto chunk = [&](const Chunks& c, int u) {
      if constexpr (kCoded) {
        const float f = __shfl(pow2_of(c.scale), srow + u * RS);
        return u32x4{decode2<T, false>(c.x[u][0], f), decode2<T, true>(c.x[u][0], f), decode2<T, false>(c.x[u][1], f),
                     decode2<T, true>(c.x[u][1], f)};
      } else {
        return c.x[u];
      }
    };
    auto whole = [&](int t, unsigned long there) { return 64 * t + 64 <= least && there == ~0ul; };
    auto store = [&](int t, unsigned long there, int buf) {
#pragma unroll
      for (int u = 0; u < PT; ++u) {
        const u32x4 x = chunk(kreg, u);
        if (sin) *reinterpret_cast<u32x4*>(ks_base + buf * G::KBUF + (srow + u * RS) * KSTR + scol) = x;
      }
      const bool look_over = !whole(t, there);
#pragma unroll
      for (int u = 0; u < PT; ++u) {
        const int row = srow + u * RS;
        u32x4 x = chunk(vreg, u);
        if (look_over) {
          unsigned any = 0;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const unsigned bad = not_finite2<T>(x[i]);
            x[i] = there >> row & 1 ? without2(x[i], bad) : 0u;
            any |= bad;
          }
          if (any && sin && (there >> row & 1)) odd[buf] = t;
        }
        if (sin) *reinterpret_cast<u32x4*>(vs_base + buf * G::VBUF + row * VSTR + scol) = x;
      }
    };

    // Table entries three tiles ahead, K and V two in registers and one in LDS: a wait for a load waits for those before
    // it too.
    PagedEntry entry = {-1, -1};
    int own = -1, own1 = -1;
    if (tid < 2) odd[tid] = -1;
    if (t0 < t1) {
      const PagedEntry first = entry_of(t0), second = entry_of(t0 + 1);
      entry = entry_of(t0 + 2);
      own = paged_row(p.c, first, w.head);
      own1 = paged_row(p.c, second, w.head);
      load(own);
    }
    X8 qf[KS];
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int c = 16 * s + 8 * hh;
      qf[s] = c < d ? *reinterpret_cast<const X8*>(qr + c) : X8{};
    }
    unsigned long there = __builtin_amdgcn_ballot_w64(own >= 0);
    __syncthreads();
    if (t0 < t1) store(t0, there, 0);
    if (t0 + 1 < t1) load(own1);
    // Q is here: told to the compiler, whose own wait for it would stand in the loop, behind the next tile's loads
    __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
    __syncthreads();

    // K (A operand of S^T): row 32 mb + n, columns 16 k + 8 hh ..
    const int koff = n * KSTR + 8 * hh;
    // V^T (A operand of O^T): the lane's transposing reads start at key 4 (g >> 1) + gi / 4, column 16 (g & 1) + 4 (gi & 3)
    const int voff = (4 * (g >> 1) + (gi >> 2)) * VSTR + 16 * (g & 1) + 4 * (gi & 3);
    const float sc = p.sc;
    float m = -INFINITY, l = 0.f;
    f32x16 o[MBO];
#pragma unroll
    for (int ob = 0; ob < MBO; ++ob) o[ob] = f32x16{};

    for (int t = t0; t < t1; ++t) {
      const int buf = (t - t0) & 1, key0 = 64 * t;
      const int own2 = paged_row(p.c, entry, w.head);
      const unsigned long there1 = __builtin_amdgcn_ballot_w64(own1 >= 0);
      const bool here = key0 < wmost;
      if (t + 1 < t1) {  // its loads have had the last tile's time to arrive
        store(t + 1, there1, buf ^ 1);
        entry = entry_of(t + 3);
        if (t + 2 < t1) load(own2);
      }
      if (here) {
        const T* kb = ks_base + buf * G::KBUF + koff;
        const T* vb = vs_base + buf * G::VBUF + voff;
        // Product i reads its K fragment kAhead products earlier; the scheduling groups hold that order (left alone, the
        // compiler reads each right before its product and waits for it)
        f32x16 s[2];
        {
          X8 kf[2 * KS];
          auto kread = [&](int i) { kf[i] = *reinterpret_cast<const X8*>(kb + 32 * (i & 1) * KSTR + 16 * (i >> 1)); };
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int i = 0; i < kAhead; ++i) kread(i);
#pragma unroll
          for (int i = 0; i < 2 * KS; ++i) {
            s[i & 1] = mma32(kf[i], qf[i >> 1], i < 2 ? f32x16{} : s[i & 1]);
            if (i + kAhead < 2 * KS) kread(i + kAhead);
          }
          __builtin_amdgcn_sched_group_barrier(0x100, kAhead, 0);
#pragma unroll
          for (int i = 0; i < 2 * KS; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            if (i + kAhead < 2 * KS) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
        auto fragment = [&](int u, int ob) {  // keys 16 u + 8 (j / 4) + 4 hh + j % 4 of columns 32 ob ..
          const T* a = vb + 16 * u * VSTR + 32 * ob;
          return join8<T>(lds_read_tr16(a), lds_read_tr16(a + 8 * VSTR));
        };
        if (key0 + 64 > wleast || there != ~0ul) {
          // shifted by the lane's part of the key, so that constants are left (the compiler would keep one key and one
          // bit a score in registers)
          const int lim = limit - key0 - 4 * hh;
          const unsigned lo = (unsigned)(there >> (4 * hh)), hi = (unsigned)(there >> 32 >> (4 * hh));
#pragma unroll
          for (int mb = 0; mb < 2; ++mb)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const int kk = 8 * (e >> 2) + (e & 3);
              s[mb][e] = 32 * mb + kk < lim && ((mb ? hi : lo) >> kk & 1) ? s[mb][e] : -INFINITY;
            }
        }
        float top = s[0][0];
#pragma unroll
        for (int mb = 0; mb < 2; ++mb)
#pragma unroll
          for (int e = 0; e < 16; ++e) top = max_nc(top, s[mb][e]);
        top = max_with_partner32(top) * sc;
        if (wave_any(top > m + kSlack)) {
          const float mn = fmaxf(m, top), alpha = exp2_fast(m - (mn == -INFINITY ? 0.f : mn));
          l *= alpha;
#pragma unroll
          for (int ob = 0; ob < MBO; ++ob) o[ob] *= alpha;
          m = mn;
        }
        const float c = m == -INFINITY ? 0.f : -m;
        X8 b[4], blo[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          float pv[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) pv[j] = exp2_fast(fmaf(s[u >> 1][8 * (u & 1) + j], sc, c));
          if constexpr (kSplitP) {
#pragma unroll
            for (int j = 0; j < 8; ++j) l += pv[j];
            split_hi_lo(pv, b[u], blo[u]);
          } else {
            b[u] = pack8(pv, (X8*)nullptr);
            typedef _Float16 h2 __attribute__((ext_vector_type(2)));
#pragma unroll
            for (int j = 0; j < 8; j += 2)
              l = __builtin_amdgcn_fdot2(h2{b[u][j], b[u][j + 1]}, h2{(f16)1.f, (f16)1.f}, l, false);
          }
        }
        // O^T += V^T P^T, each fragment read kAhead products earlier
        {
          X8 vf[4 * MBO];
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int i = 0; i < kAhead; ++i) vf[i] = fragment(i / MBO, i % MBO);
#pragma unroll
          for (int i = 0; i < 4 * MBO; ++i) {
            o[i % MBO] = mma32(vf[i], b[i / MBO], o[i % MBO]);
            if constexpr (kSplitP) o[i % MBO] = mma32(vf[i], blo[i / MBO], o[i % MBO]);
            if (i + kAhead < 4 * MBO) vf[i + kAhead] = fragment((i + kAhead) / MBO, (i + kAhead) % MBO);
          }
          __builtin_amdgcn_sched_group_barrier(0x100, 2 * kAhead, 0);
#pragma unroll
          for (int i = 0; i < 4 * MBO; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x008, kSplitP ? 2 : 1, 0);
            if (i + kAhead < 4 * MBO) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
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
      own = own1;
      own1 = own2;
      there = there1;
      // the workgroup's LDS is in order; loads on their way into registers stay on it (__syncthreads would wait for them)
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
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
      if (p.nsplit > 1 && hh == 0) *reinterpret_cast<float2*>(p.ml + 2 * part) = direct ? float2{0.f, -1.f} : float2{m, l};
    }
    __syncthreads();  // the next rows' first tile replaces buffer 0
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
