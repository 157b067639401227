// Host-side launch interface of the cache in 8 bits and of beam search, between cats_api_cache.hip and cats_inst_kv8.hip (compiled once
// per dtype).
#pragma once
#include "cats_beam.h"
#include "cats_kv8.h"
#include "cats_launch.h"

namespace cats {

// The cache in 8 bits (cats_kv8.h), 16-bit types.  launch_kv8_attn fills in what the plan decides.
struct KvAttnPlan {
  bool prompt; // kv8_attn_prompt_kernel
  int splits;  // of a row's cache
  bool seal;   // the new tokens are in the tails only: quantise the blocks they complete
};
KvAttnPlan kv8_attn_plan(int B, int T, int heads, int kv_heads, int blocks, int window);
template <class DT>
hipError_t launch_kv8_append(int D, const KvAppendArgs& a, int B, hipStream_t stream);
template <class DT>
hipError_t launch_kv8_attn(int D, const KvAttnPlan& plan, KvAttnArgs a, hipStream_t stream);

// The pass over the logits of beam search (cats_beam.h): 8 or 32 elements a lane.
template <class DT>
hipError_t launch_beam_rows(int per_lane, const BeamArgs& a, int rows, hipStream_t stream);

}  // namespace cats
