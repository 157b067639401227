// Host-side launch interface of the cache of pages and of packed attention, between cats_api_paged.hip and cats_inst_paged.hip (compiled once
// per dtype).
#pragma once
#include "cats_launch.h"
#include "cats_packed.h"

namespace cats {

template <class DT>
hipError_t launch_paged_append(int D, bool wide, const PagedAppendArgs& a, hipStream_t stream);

// Which kernel attention over pages takes, and into how many parts it splits keys.
struct PackedPlan {
  bool tiles, group_tiles;   // packed_attn_tiles_kernel, and not packed_attn_step_kernel, for a sequence's own keys, and for those that its group shares
  int splits, group_splits;  // 0: none are shared
};
// plan NULL: keys and values of the call.  launch_packed_attn fills in what the plan decides.
template <class DT>
hipError_t launch_packed_attn(int D, const PackedPlan* plan, PackedAttnArgs a, hipStream_t stream);

}  // namespace cats
