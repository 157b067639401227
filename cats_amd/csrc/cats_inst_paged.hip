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
    if (!plan || !plan->step) {
      a.slots = packed_slots(a.seq.N, a.seq.B + 2, a.group, kTileRows);
      const int all = a.seq.N * a.group / kTileRows * a.kv_heads, cus = current_device_cus();
      a.turn = all <= 2 * cus && all > cus ? cus : INT_MAX;
      return launch_kernel(plan ? packed_attn_tiles_kernel<CATS_DT, HD, true> : packed_attn_tiles_kernel<CATS_DT, HD, false>, dim3(a.slots * a.kv_heads), dim3(256), 0,
                           stream, a);
    }
    a.splits = plan->splits;
    a.group_splits = plan->group_splits;
    a.slots = packed_slots(a.seq.N, a.seq.B + 2, a.group, kStepBlock);
    a.group_slots = a.group_splits ? packed_slots(a.seq.N, a.seq.B / a.members + 2, a.group, kStepBlock) : 0;
    a.by_splits = divisor(a.splits);
    a.by_group_splits = divisor(a.group_splits > 0 ? a.group_splits : 1);
    hipError_t e = launch_kernel(packed_attn_step_kernel<CATS_DT, HD>, dim3((a.slots * a.splits + a.group_slots * a.group_splits) * a.kv_heads), dim3(256), 0, stream, a);
    if (e != hipSuccess || a.splits + a.group_splits == 1) return e;
    const long long rows = (long long)a.seq.N * a.kv_heads * a.group;
    if (a.splits + a.group_splits > 8) return launch_kernel(packed_join_kernel<CATS_DT, HD, true>, dim3((unsigned)rows), dim3(256), 0, stream, a);
    return launch_kernel(packed_join_kernel<CATS_DT, HD, false>, dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, stream, a);
  });
}

}  // namespace cats
