// Host-side launch interface of the cache of pages and of packed attention, between cats_api_paged.hip and cats_inst_paged.hip (compiled once
// per dtype).
#pragma once
#include "cats_launch.h"
#include "cats_packed.h"

namespace cats {

template <class DT>
hipError_t launch_paged_append(int D, bool wide, const PagedAppendArgs& a, hipStream_t stream);
template <class DT>
hipError_t launch_packed_attn(int D, bool paged, PackedAttnArgs a, hipStream_t stream);

}  // namespace cats
