// Attention over a cache in 8 bits (16-bit types) and the selection of beam search for one dtype.  Compiled three times
// (-DCATS_DT=F16 / BF16 / F32), beside cats_inst.hip.
#include <type_traits>

#include "cats_launch_cache.h"

#ifndef CATS_DT
#error "compile with -DCATS_DT=F16|BF16|F32"
#endif

namespace cats {

namespace {

template <class DT>
struct KvLaunch {
  template <int D>
  static hipError_t append_d(const KvAppendArgs& a, int B, hipStream_t stream) {
    // the blocks that T tokens touch at most, wherever they start
    const dim3 grid((a.T + kKvBlock - 2) / kKvBlock + 1, a.c.heads, B);
    return launch_kernel(kv8_append_kernel<DT, D>, grid, dim3(256), 0, stream, a);
  }
  static hipError_t append(int D, const KvAppendArgs& a, int B, hipStream_t stream) {
    switch (D) {
      case 32: return append_d<32>(a, B, stream);
      case 64: return append_d<64>(a, B, stream);
      case 128: return append_d<128>(a, B, stream);
      case 256: return append_d<256>(a, B, stream);
    }
    return hipErrorInvalidValue;
  }
  // A workgroup a row from five splits on.  A row per group of lanes / a workgroup, with attention, in us, heads of 128: 2 splits, 32 rows of 32 heads
  // 28.8 / 29.4; 8 splits, 8 rows 27.5 / 27.1; 32 splits of 20 rows of 14 heads of 64 21.1 / 20.5; 4 splits, 16 rows the same.
  template <int D, int ROWS, int UNIT>
  static hipError_t join(const KvAttnArgs& a, hipStream_t stream) {
    const int items = a.pairs * a.T * a.group, per = 256 / (D / 4);
    if (a.splits > 4) return launch_kernel(kv8_join_kernel<DT, D, ROWS, UNIT, true>, dim3(items), dim3(256), 0, stream, a);
    return launch_kernel(kv8_join_kernel<DT, D, ROWS, UNIT, false>, dim3((items + per - 1) / per), dim3(256), 0, stream, a);
  }
  template <int D>
  static hipError_t attn_d(const KvAttnPlan& plan, const KvAttnArgs& a, hipStream_t stream) {
    const int rows = a.T * a.group;
    if (plan.prompt) {
      const dim3 grid(a.pairs, (rows + kKvPromptRows - 1) / kKvPromptRows, a.splits);
      hipError_t e = launch_kernel(kv8_attn_prompt_kernel<DT, D>, grid, dim3(256), 0, stream, a);
      return e == hipSuccess && a.splits > 1 ? join<D, kKvPromptRows, kKvPromptUnit>(a, stream) : e;
    }
    auto kern = plan.seal                   ? kv8_attn_step_kernel<DT, D, false, true>
                : a.T > 1 || a.window ? kv8_attn_step_kernel<DT, D, true, false>
                                      : kv8_attn_step_kernel<DT, D, false, false>;
    hipError_t e = launch_kernel(kern, dim3(a.pairs, a.splits + plan.seal, (rows + 15) / 16), dim3(256), 0, stream, a);
    return e == hipSuccess && a.splits > 1 ? join<D, 16, kKvStepWaves>(a, stream) : e;
  }
  static hipError_t attn(int D, const KvAttnPlan& plan, const KvAttnArgs& a, hipStream_t stream) {
    switch (D) {
      case 32: return attn_d<32>(plan, a, stream);
      case 64: return attn_d<64>(plan, a, stream);
      case 128: return attn_d<128>(plan, a, stream);
      case 256: return attn_d<256>(plan, a, stream);
    }
    return hipErrorInvalidValue;
  }
};
template <>
struct KvLaunch<F32> {
  static hipError_t append(int, const KvAppendArgs&, int, hipStream_t) { return hipErrorInvalidValue; }
  static hipError_t attn(int, const KvAttnPlan&, const KvAttnArgs&, hipStream_t) { return hipErrorInvalidValue; }
};

}  // namespace

template <>
hipError_t launch_kv8_append<CATS_DT>(int D, const KvAppendArgs& a, int B, hipStream_t stream) {
  return KvLaunch<CATS_DT>::append(D, a, B, stream);
}

template <>
hipError_t launch_kv8_attn<CATS_DT>(int D, const KvAttnPlan& plan, KvAttnArgs a, hipStream_t stream) {
  a.splits = plan.splits;
  return KvLaunch<CATS_DT>::attn(D, plan, a, stream);
}

template <>
hipError_t launch_beam_rows<CATS_DT>(int per_lane, const BeamArgs& a, int rows, hipStream_t stream) {
  auto kern = per_lane == 8 ? beam_rows_kernel<CATS_DT, 8> : beam_rows_kernel<CATS_DT, 32>;
  return launch_kernel(kern, dim3(a.pieces, rows), dim3(256), 0, stream, a);
}

}  // namespace cats
