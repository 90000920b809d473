// Which kernel runs a paged-attention call, with how many rows a tile and how many key splits.
#include <algorithm>

#include "paged.hpp"

namespace samhip {

PagedPlan paged_plan(int dtype, int cache_dtype, int tokens, int batch, int heads, int kv_heads, int d, int max_q,
                     int max_len, int cus) {
  (void)cache_dtype;
  PagedPlan plan = {};
  const long group = heads / kv_heads, rows = (long)std::max(std::min(max_q, tokens), 1) * group;
  plan.many = dtype != kF32 && rows > 32;
  plan.rows = plan.many ? 128 : rows <= 16 || d > 128 ? 16 : 32;
  // a workgroup goes on to further tiles: where max_q is far above most chunks, a million of them do
  const long units = (long)kv_heads * batch, cap = std::max(1L, (1L << 20) / units);
  plan.rtiles = (int)std::min((rows + plan.rows - 1) / plan.rows, cap);
  const long base = plan.rtiles * units;
  if (plan.many) {
    // as many workgroups as run at once (three a CU up to head dim 64, two to 128, one past it), with four tiles of 64
    // keys a split at least
    const long slots = (d > 128 ? 1L : d > 64 ? 2L : 3L) * cus, most = ((long)max_len + 255) / 256;
    plan.nsplit = (int)std::max(1L, std::min(std::min(slots / base, most), 64L));
  } else {
    // eight workgroups a CU, if every split then has eight blocks of 32 keys for each of its four waves
    const long want = (8L * cus + base - 1) / base, most = ((long)max_len + 1023) / 1024;
    plan.nsplit = (int)std::max(1L, std::min(std::min(want, most), 256L));
  }
  if ((long)tokens * heads * (d / 4) >= 1L << 32) plan.nsplit = 1;  // more than the joining launch has threads for
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
  hipError_t e = dtype == kF32 ? paged_f32(cache_dtype, p, plan.rows, stream)
                 : plan.many   ? paged_many(dtype, cache_dtype, p, stream)
                               : paged_few(dtype, cache_dtype, p, plan.rows, stream);
  if (e == hipSuccess && p.nsplit > 1) e = paged_combine(dtype, p, stream);
  return e;
}

}  // namespace samhip
