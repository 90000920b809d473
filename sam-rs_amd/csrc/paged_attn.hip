// Which kernel runs a paged-attention call, with how many rows a tile and how many key splits.
#include <algorithm>

#include "paged.hpp"

namespace samhip {

// Key splits of a call bound by f32 products, `base` workgroups of which `slots` run at once: the fewest rounds, where a
// split costs 5% more. 2048 rows over 4096 keys, 8 heads of 128 (two whole rounds), 401, 425, 468 and 550 us with 1, 2, 4 and
// 8 splits; 41 chunks of 125 rows over 4320 keys, one head, at 256 (1.3 rounds) 605, 491, 473 and 547 with 1 to 4, at 96 (0.6)
// 169, 183, 138 and 157; 9 with 8 heads of 128 (1.1) 374, 304, 301 and 301.
static long f32_splits(long base, long slots) {
  long best = 1;
  auto cost = [&](long n) { return (double)((base * n + slots - 1) / slots) / n * (1 + 0.05 * (n - 1)); };
  for (long n = 2; n <= 64; ++n)
    if (cost(n) < cost(best)) best = n;
  return best;
}

PagedPlan paged_plan(int dtype, int cache_dtype, int tokens, int batch, int heads, int kv_heads, int d, int max_q,
                     int max_len, int cus) {
  PagedPlan plan = {};
  const long group = heads / kv_heads, rows = (long)std::max(std::min(max_q, tokens), 1) * group;
  // The many-row kernel past 32 rows a key head, which the other takes in two passes over the keys: 8 sequences of 8192, 8
  // heads of 128 in f16, 33 rows each 56 against 110 us, 32 rows 55 against 62; at 64 42 against 52 and 41 against 35; 4 of 4
  // heads of 256, 54 against 69 and 53 against 42; one of 65536 with 2 heads of 128 35 against 29 and 33 against 28 (the rule
  // counts rows alone, so this one call loses).
  plan.many = dtype != kF32 && rows > 32;
  // 32 rows a tile above 16 where registers allow it: the first of these calls at 17 rows 61 us against 90 with two tiles of
  // 16, the third (which they do not) 42
  plan.rows = plan.many ? 128 : rows <= 16 || d > 128 ? 16 : 32;
  // a workgroup goes on to further tiles: where max_q is far above most chunks, a million of them do
  const long units = (long)kv_heads * batch, cap = std::max(1L, (1L << 20) / units);
  plan.rtiles = (int)std::min((rows + plan.rows - 1) / plan.rows, cap);
  const long base = plan.rtiles * units;
  if (plan.many) {
    // As many workgroups as run at once (three a CU up to head dim 64, two to 128, one past it), with four tiles of 64
    // keys a split at least. More only add partial results: six sequences of up to 7000 keys, 8 heads of 64, 1024 rows each,
    // 155, 113, 115 and 120 us with 1, 2, 3 and 4 splits; 4096 rows over 28736 keys, 256, 229 and 315 with 8 and 16.
    const long slots = (d > 128 ? 1L : d > 64 ? 2L : 3L) * cus, full = std::min(slots / base, max_len / 256L);
    // Up to eight of a tile each while they are one a CU: 100 rows over 1000 keys, 8 heads of 64, 22, 13 and 12 us with 1, 4
    // and 8, 64 over 500, 8 heads of 128, 18, 13 and 11; 1000 over 1000, 8 heads of 64, 23, 16 and 18.
    const long small = max_len >= 384 ? std::min(std::min(cus / base, max_len / 64L), 8L) : 1;
    plan.nsplit = (int)std::max(1L, std::min(std::max(full, small), 64L));
    // more than eight are joined in a loop: 1000 rows over 3000 keys, 2 key heads of 128, 27 us with 8, 31 with 12, 30 with 16
    if (plan.nsplit > 8 && plan.nsplit < 16) plan.nsplit = 8;
  } else {
    // Four workgroups a CU (two past head dim 128, where one runs at a time), so that sequences of different lengths share
    // the card, of 512 KB of keys and values each at least. 32 sequences, 8 key heads of 128 in e4m3: 820 to 8192 keys 92, 94,
    // 80, 84, 83 and 96 us with 2, 3, 4, 6, 8 and 12 splits, 8192 each 118, 118, 121, 125, 134 and 148; 4 heads of 256 in e4m3,
    // 8192 each, 103, 112 and 132 with 2, 4 and 8. Calls that f32 products bound count rounds.
    const long bytes = 2L * d * (cache_dtype == kE4M3 ? 1 : dtype == kF32 ? 4 : 2) * max_len;  // a sequence's, of one head
    const long want = plan.rtiles > 1 && dtype == kF32 ? f32_splits(base, (d > 64 ? 1L : 2L) * cus)
                                                       : ((d > 128 ? 2L : 4L) * cus + base - 1) / base;
    const long many = std::min(want, bytes >> 19);
    // One a CU, of 128 KB each at least: a CU alone reads 60 GB/s. In f16, 2048 keys of 4 heads of 128 take 22.6, 16.4, 12.2 and
    // 10.3 us with 1, 2, 4 and 8 splits, 4096 of 4 heads of 64 25.4, 17.2, 11.9 and 9.6, 1024 of 8 heads of 128 14.0, 11.7 and
    // 9.7 with 1, 2 and 4. Below 448 KB the second launch costs what it gains (577 keys of 8 heads of 64 8.0 and 8.1 with 1
    // and 4, without the host's 3 us).
    const long few = bytes > 448 << 10 ? std::min(cus / base, (bytes + (1 << 17) - 1) >> 17) : 1;
    plan.nsplit = (int)std::min(std::max(std::max(many, few), 1L), 256L);
  }
  // no more threads for the launch that joins the splits than 32 bits count: d / 4 a row to 8 splits, 512 for 32 columns past
  if ((long)tokens * heads * ((d + 31) / 32) >= 1L << 23) plan.nsplit = std::min(plan.nsplit, 8);
  if ((long)tokens * heads * (d / 4) >= 1L << 32) plan.nsplit = 1;
  plan.round = (int)(cus / (units * plan.nsplit));
  const long blocks = ((long)max_len + 31) / 32;
  plan.per = (int)std::min((blocks + plan.nsplit - 1) / plan.nsplit, 1L << 26);
  if (plan.nsplit > 1) {
    plan.part_bytes = (long)plan.nsplit * tokens * heads * d * 4;
    plan.total = plan.part_bytes + (long)plan.nsplit * tokens * heads * 8;
  }
  return plan;
}

hipError_t paged_attention(int dtype, int cache_dtype, PagedParams p, const PagedPlan& plan, hipStream_t stream) {
  p.rtiles = plan.rtiles;
  p.nsplit = plan.nsplit;
  p.per = plan.per;
  p.round = plan.round;
  hipError_t e = dtype == kF32 ? paged_f32(cache_dtype, p, plan.rows, stream)
                 : plan.many   ? paged_many(dtype, cache_dtype, p, stream)
                               : paged_few(dtype, cache_dtype, p, plan.rows, stream);
  if (e == hipSuccess && p.nsplit > 1) e = paged_combine(dtype, p, stream);
  return e;
}

}  // namespace samhip
