// The cache of pages and packed attention for one dtype.  Compiled twice (-DCATS_DT=F16 / BF16).
#include "cats_launch_paged.h"

#ifndef CATS_DT
#error "compile with -DCATS_DT=F16|BF16"
#endif

namespace cats {
namespace {

template <class F>
hipError_t for_head_dim(int D, F f) {
  switch (D) {
    case 32: return f(std::integral_constant<int, 32>());
    case 64: return f(std::integral_constant<int, 64>());
    case 128: return f(std::integral_constant<int, 128>());
    case 256: return f(std::integral_constant<int, 256>());
  }
  return hipErrorInvalidValue;
}

}  // namespace

template <>
hipError_t launch_paged_append<CATS_DT>(int D, bool wide, const PagedAppendArgs& a, hipStream_t stream) {
  return for_head_dim(D, [&](auto d) {
    constexpr int HD = decltype(d)::value;
    const int units = (a.heads + 2 * a.pool.heads) * (HD / 16), blocks = (units + 511) / 512, threads = ((units + blocks - 1) / blocks + 63) / 64 * 64;
    const dim3 grid((a.seq.N + a.per - 1) / a.per, blocks);
    return launch_kernel(wide ? paged_append_kernel<CATS_DT, HD, true> : paged_append_kernel<CATS_DT, HD, false>, grid, dim3(threads), 0, stream, a);
  });
}

template <>
hipError_t launch_packed_attn<CATS_DT>(int D, const PackedPlan* plan, PackedAttnArgs a, hipStream_t stream) {
  return for_head_dim(D, [&](auto d) {
    constexpr int HD = decltype(d)::value;
    a.by_group = divisor(a.group);
    a.by_heads = divisor(a.kv_heads);
    a.by_members = divisor(a.members > 0 ? a.members : 1);
    const int N = a.seq.N, B = a.seq.B;
    if (!plan || (plan->tiles && plan->splits + plan->group_splits == 1)) {
      a.slots = packed_slots(N, B + 2, a.group, kTileRows);
      a.cus = current_device_cus();
      return launch_kernel(plan ? packed_attn_tiles_kernel<CATS_DT, HD, PAGES> : packed_attn_tiles_kernel<CATS_DT, HD, PROMPT>, dim3(a.slots * a.kv_heads), dim3(256), 0,
                           stream, a);
    }
    a.splits = plan->splits;
    a.group_splits = plan->group_splits;
    a.by_splits = divisor(a.splits);
    a.by_group_splits = divisor(a.group_splits > 0 ? a.group_splits : 1);
    const int rows_of[2] = {kStepRows, kTileRows};
    a.group_blocks = a.group_splits ? a.group_splits * packed_slots(N, B / a.members + 2, a.group, rows_of[plan->group_tiles]) : 0;
    const dim3 grid((a.group_blocks + a.splits * packed_slots(N, B + 2, a.group, rows_of[plan->tiles])) * a.kv_heads);
    const hipError_t e = launch_kernel(plan->tiles         ? packed_attn_tiles_kernel<CATS_DT, HD, SPLIT>
                                       : plan->group_tiles ? packed_attn_both_kernel<CATS_DT, HD>
                                                           : packed_attn_step_kernel<CATS_DT, HD>,
                                       grid, dim3(256), 0, stream, a);
    if (e != hipSuccess || a.splits + a.group_splits == 1) return e;
    const long long rows = (long long)a.seq.N * a.kv_heads * a.group;
    if (a.splits + a.group_splits > 8) return launch_kernel(packed_join_kernel<CATS_DT, HD, true>, dim3((unsigned)rows), dim3(256), 0, stream, a);
    return launch_kernel(packed_join_kernel<CATS_DT, HD, false>, dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, stream, a);
  });
}

}  // namespace cats
