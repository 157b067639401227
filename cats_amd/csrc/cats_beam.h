// Beam search on the device: the best continuations of every group of beams, and the caches moved to the beams that go on.
#pragma once
#include "cats_device.h"

namespace cats {

constexpr int kBeamMax = 16;  // beams of a group, before and after

// ---- selection ---------------------------------------------------------------------------------------------------------------------
//   total(b, v) = score[b] + logit[b][v] - log(sum over v of exp(logit[b][v]));   the best `keep` of a group, ties to the lowest b * V + v
// A beam that has finished goes on only as (b, eos) with its score.  Totals that are not finite count as -infinity.
//
// beam_rows_kernel: one pass over the logits.  A workgroup holds 256 E of them in registers and leaves their maximum, the sum of exponentials and
// the best `keep`.  For those: of the 64 sets of values that lane l of each wave holds, the keep-th best of their best values bounds what can be
// among them, so what is not below it is gathered (some more than `keep`) and ranked by comparing each with all; only where ties make that
// more than 64 are each wave's best taken one by one and joined.  beam_join_kernel: a workgroup per group, a wave per beam joins its row's pieces in the same way, and
// the beams' candidates are ranked by their totals in 64 bits: the order has to be that of the sums, which differ in their last bits only.
// A row with a NaN or +infinity has no finite total at all, so neither has to be found among the best.
// 16 groups of 16 beams, 100003 words in 32 bits: 19.6 us, 5.2 TB/s where a read stream reaches 7.1, and 9.2 for the join, whose sixteen waves share a CU.
// 32 elements a lane with six waves a SIMD; a bound a wave instead of a workgroup 30.3 us, 64 elements 21 to 26.  4 beams of 32000 words: 4.4 and 4.9 us.

struct BeamArgs {
  const void* logits;     // rows of V, row_stride elements apart
  long long row_stride;
  const float* scores;    // (groups, beams)
  const uint8_t* finished;
  long long eos;
  float* scores_out;      // (groups, keep)
  int64_t* parents_out;
  int64_t* tokens_out;
  uint8_t* finished_out;
  float* ml;              // [row][piece][2] maximum and sum of exponentials
  float* vals;            // [row][piece][keep], in order
  int* ids;               // -1: none
  int beams, V, keep, pieces;
};

template <int CTRL>
__device__ __forceinline__ float dpp_get(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
template <int CTRL>
__device__ __forceinline__ float dpp_max(float v) { return fmaxf(v, dpp_get<CTRL>(v)); }
// Largest over the 64 lanes, the same in all; the steps of wave_sum.
__device__ __forceinline__ float wave_max(float v) {
  v = dpp_max<0xB1>(v);
  v = dpp_max<0x4E>(v);
  v = dpp_max<0x141>(v);
  v = dpp_max<0x140>(v);
  const int i = __float_as_int(v);
  return fmaxf(fmaxf(__int_as_float(__builtin_amdgcn_readlane(i, 0)), __int_as_float(__builtin_amdgcn_readlane(i, 16))),
               fmaxf(__int_as_float(__builtin_amdgcn_readlane(i, 32)), __int_as_float(__builtin_amdgcn_readlane(i, 48))));
}
// The k-th largest of the 64 lanes' values, k in 1..16, the same in all.  Rows of 16 lanes are sorted in descending order (a bitonic sort whose every
// merge starts with a mirrored exchange); of two sorted rows, the larger of each lane and its mirrored one are the 16 largest, in bitonic order.
// Some 60 instructions, where taking the largest k times is 30 each.
__device__ __forceinline__ float wave_kth(float v, int k, int lane) {
  auto order = [&](float other, int bit) {  // the lower lane of a pair keeps the larger value
    const float hi = fmaxf(v, other), lo = fminf(v, other);
    v = lane & bit ? lo : hi;
  };
  auto merge = [&]() {  // of a bitonic row
    order(dpp_get<0x128>(v), 8);
    order(dpp_get<0x1B>(dpp_get<0x141>(v)), 4);
    order(dpp_get<0x4E>(v), 2);
    order(dpp_get<0xB1>(v), 1);
  };
  order(dpp_get<0xB1>(v), 1);
  order(dpp_get<0x1B>(v), 2);
  order(dpp_get<0xB1>(v), 1);
  order(dpp_get<0x141>(v), 4);
  order(dpp_get<0x4E>(v), 2);
  order(dpp_get<0xB1>(v), 1);
  order(dpp_get<0x140>(v), 8);
  order(dpp_get<0x1B>(dpp_get<0x141>(v)), 4);
  order(dpp_get<0x4E>(v), 2);
  order(dpp_get<0xB1>(v), 1);
  v = fmaxf(v, __shfl_xor(v, 31, kWave));
  merge();
  v = fmaxf(v, __shfl_xor(v, 47, kWave));
  merge();
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), k - 1));
}
// Floats ordered as unsigned integers, -0 as 0.
__device__ __forceinline__ uint32_t beam_key(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return b >> 31 ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ int wave_min(int v) {
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) v = min(v, __shfl_xor(v, o, kWave));
  return v;
}
// LDS of this wave alone: what its lanes have written is there for all of them.
__device__ __forceinline__ void wave_lds_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup", "local");
  __builtin_amdgcn_wave_barrier();
}

struct BeamList {  // in LDS, of a wave
  float val[kWave];
  int id[kWave];
};

// Writes the best `keep` of the `count` <= 64 pairs that the lanes hold to `best`, in order, lower ids first among equal values.
__device__ __forceinline__ void wave_rank(float v, int n, int count, int keep, int lane, BeamList& best) {
  const uint32_t hi = beam_key(v), lo = ~(uint32_t)n;  // larger is better
  const uint64_t mine = (uint64_t)hi << 32 | lo;
  int rank = 0;
  for (int j = 0; j < count; j++) {
    const uint64_t other = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)hi, j) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)lo, j);
    rank += other > mine;
  }
  if (lane < count && rank < keep) {
    best.val[rank] = v;
    best.id[rank] = n;
  }
}
// The same of any number of values, taken one by one: for those with many equal ones.  `own` is what id() computes from, hidden from the compiler
// in every round: E ids kept for this would take the registers that let more waves wait for memory.
template <int E, class Id>
__device__ __forceinline__ void wave_pick(const float (&x)[E], Id id, int& own, int keep, int lane, BeamList& best) {
  uint64_t gone = 0;  // of this lane's values
  static_assert(E <= 64, "a bit each");
  for (int k = 0; k < keep; k++) {
    asm volatile("" : "+v"(own));
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < E; i++) top = gone >> i & 1 ? top : fmaxf(top, x[i]);
    top = wave_max(top);
    int first = INT32_MAX, which = 0;
#pragma unroll
    for (int i = 0; i < E; i++) {
      const int n = id(i);
      const bool in = !(gone >> i & 1) && n >= 0 && x[i] == top && n < first;
      first = in ? n : first;
      which = in ? i : which;
    }
    const int lowest = wave_min(first);
    if (lowest == INT32_MAX) break;
    if (first == lowest) gone |= (uint64_t)1 << which;
    if (lane == 0) {
      best.val[k] = top;
      best.id[k] = lowest;
    }
  }
}
// Appends a value of each lane that is `in` to the list, as far as it has room; the count goes on.
__device__ __forceinline__ void wave_take(bool in, float v, int n, int& count, BeamList& list) {
  const uint64_t b = __ballot(in);
  const int at = count + ballot_rank(b);
  if (in && at < kWave) {
    list.val[at] = v;
    list.id[at] = n;
  }
  count += __popcll(b);
}

// Writes the best `keep` of the wave's values to `best`, in order, lower ids first among equal ones, ids of -1 behind the last.  id(i) is that of
// x[i], -1 for no entry (and x[i] = -infinity).  The lowest 32 ids of the wave,
// or all, are within the first FRONT values.
template <int FRONT, int E, class Id>
__device__ __forceinline__ void wave_best(const float (&x)[E], Id id, int keep, int lane, BeamList& list, BeamList& best) {
  float bound = -INFINITY;
  if constexpr (E > 1) {  // one value a lane fits the list as it is
    float mine = -INFINITY;
#pragma unroll
    for (int i = 0; i < E; i++) mine = fmaxf(mine, x[i]);
    bound = wave_kth(mine, keep, lane);
  }
  int count = 0;
  const bool low = bound == -INFINITY;  // less than `keep` lanes have more than that, or there is one value a lane
#pragma unroll
  for (int i = 0; i < E; i++) {
    const bool in = low ? x[i] > bound : x[i] >= bound;
    if (__any(in)) wave_take(in, x[i], id(i), count, list);
  }
  if (low && count < keep) {  // then values of -infinity are among the best, those with the lowest ids
#pragma unroll
    for (int i = 0; i < FRONT; i++) wave_take(x[i] == -INFINITY && id(i) >= 0, x[i], id(i), count, list);
  }
  if (lane < keep) best.id[lane] = -1;
  wave_lds_sync();
  int none = 0;
  if (count <= kWave) wave_rank(lane < count ? list.val[lane] : 0.f, lane < count ? list.id[lane] : 0, count, keep, lane, best);
  else wave_pick(x, id, none, keep, lane, best);
  wave_lds_sync();
}

typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));  // wherever an element starts

template <class DT, int E>
__global__ __launch_bounds__(256, 6) void beam_rows_kernel(BeamArgs p) {
  typedef typename DT::st st;
  constexpr int VEC = DT::VEC, W = 4, G = E / VEC;
  __shared__ BeamList s_list[W], s_best[W];
  __shared__ float s_max[W][kWave], s_sum[W];
  __shared__ int s_count[W];
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x >> 6, row = blockIdx.y, piece = blockIdx.x;
  if (p.finished && p.finished[row]) return;
  const st* x = (const st*)p.logits + row * p.row_stride;
  // The wave's elements, in vectors of VEC that go round the lanes, wherever the row starts: which words are summed together goes by their ids alone, so rows
  // that are the same have the same sums to the bit, and tie.
  const int first = (piece * W + wave) * kWave * E;
  float val[E];
  int own = first + lane * VEC;
  auto id = [&](int i) {
    const int at = own + i / VEC * kWave * VEC + i % VEC;
    return at < p.V ? at : -1;
  };
  if (first + kWave * E <= p.V) {
    u32x4 w[G];
#pragma unroll
    for (int i = 0; i < G; i++) w[i] = __builtin_nontemporal_load((const u32x4_any*)(x + first + (i * kWave + lane) * VEC));
#pragma unroll
    for (int i = 0; i < E; i++) {
      const uint32_t c = w[i / VEC][i % VEC * 4 / VEC];
      if constexpr (VEC == 4) val[i] = __uint_as_float(c);
      else val[i] = DT::tof((st)(c >> (16 * (i & 1))));
    }
  } else {
    st w[E];
#pragma unroll
    for (int i = 0; i < E; i++) w[i] = x[max(id(i), 0)];
#pragma unroll
    for (int i = 0; i < E; i++) val[i] = id(i) >= 0 ? DT::tof(w[i]) : -INFINITY;
  }
  float top[G], most = -INFINITY;
#pragma unroll
  for (int g = 0; g < G; g++) {
    top[g] = val[g * VEC];
#pragma unroll
    for (int i = 1; i < VEC; i++) top[g] = fmaxf(top[g], val[g * VEC + i]);
    most = fmaxf(most, top[g]);
  }
  s_max[wave][lane] = most;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < W; w++) most = fmaxf(most, s_max[w][lane]);
  const float m = wave_max(most), bound = wave_kth(most, p.keep, lane);
  // exp of a difference that is rounded once: within 2^-24 of |x - m|, as the difference itself is
  const float base = m == -INFINITY ? 0.f : m;
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < E; i++) sum += __builtin_amdgcn_exp2f((val[i] - base) * 1.44269504088896341f);
  sum = wave_sum(sum);
  const bool low = bound == -INFINITY;  // less than `keep` of the 64 have more than that
  int count = 0;
#pragma unroll
  for (int g = 0; g < G; g++) {
    if (!__any(top[g] >= bound)) continue;
#pragma unroll
    for (int i = g * VEC; i < (g + 1) * VEC; i++) {
      const bool in = low ? val[i] > bound : val[i] >= bound;
      if (__any(in)) wave_take(in, val[i], id(i), count, s_list[wave]);
    }
  }
  if (lane == 0) {
    s_count[wave] = count;
    s_sum[wave] = sum;
  }
  __syncthreads();
  int counts[W], all = 0;
#pragma unroll
  for (int w = 0; w < W; w++) all += counts[w] = s_count[w];
  float v = -INFINITY;
  int n = -1;
  if (all <= kWave) {
    if (wave != 0) return;
    if (low && all < p.keep) {  // then values of -infinity are among the best, those with the lowest ids: in the first lanes' first vectors
#pragma unroll
      for (int i = 0; i < VEC; i++) wave_take(lane < 32 / VEC && val[i] == -INFINITY && id(i) >= 0, val[i], id(i), counts[0], s_list[0]);
      all = counts[0] + counts[1] + counts[2] + counts[3];
    }
    if (lane < p.keep) s_best[0].id[lane] = -1;
    wave_lds_sync();
    int w = 0, at = lane;
#pragma unroll
    for (int i = 0; i < W - 1; i++) {
      const bool on = w == i && at >= counts[i];
      at -= on ? counts[i] : 0;
      w += on;
    }
    if (lane < all) v = s_list[w].val[at], n = s_list[w].id[at];
  } else {
    BeamList& best = s_best[wave];
    if (lane < p.keep) best.id[lane] = -1;
    wave_lds_sync();
    if (count <= kWave) wave_rank(lane < count ? s_list[wave].val[lane] : 0.f, lane < count ? s_list[wave].id[lane] : 0, count, p.keep, lane, best);
    else wave_pick(val, id, own, p.keep, lane, best);
    __syncthreads();
    if (wave != 0) return;
    const int from = lane / p.keep, which = lane - from * p.keep;
    v = from < W ? s_best[from < W ? from : 0].val[which] : 0.f;
    n = from < W ? s_best[from < W ? from : 0].id[which] : -1;
    wave_lds_sync();
    all = 0;
    wave_take(n >= 0, v, n, all, s_list[0]);
    if (lane < p.keep) s_best[0].id[lane] = -1;
    wave_lds_sync();
    if (lane < all) v = s_list[0].val[lane], n = s_list[0].id[lane];
  }
  wave_rank(v, n, all, p.keep, lane, s_best[0]);
  wave_lds_sync();
  const size_t out = (size_t)row * p.pieces + piece;
  if (lane < p.keep) {
    p.vals[out * p.keep + lane] = s_best[0].val[lane];
    p.ids[out * p.keep + lane] = s_best[0].id[lane];
  }
  if (lane == 0) {
    p.ml[2 * out] = m;
    p.ml[2 * out + 1] = s_sum[0] + s_sum[1] + s_sum[2] + s_sum[3];
  }
}

// Doubles ordered as unsigned integers, -0 as 0.  0 is below them all.
__device__ __forceinline__ uint64_t beam_key(double x) {
  const uint64_t b = (uint64_t)__double_as_longlong(x + 0.0);
  return b >> 63 ? ~b : b | 1ull << 63;
}

// Candidates of a row come in pieces of `keep`; a wave takes 256 at a time beside the best it has (512: 16 beams of 32000 words 15.3 us, 14.7; of 200000
// 27.0, 25.9).  What the beams offer is in order for each of them
// (total, then id), so of equal totals the earlier offer is the better one.  Few of them are ranked in 64 bits: those whose totals, rounded to
// float, which keeps their order, are not below the keep-th best of the lanes'.
template <int N>
__global__ __launch_bounds__(N* kWave) void beam_join_kernel(BeamArgs p) {
  __shared__ BeamList s_list[N], s_best[N];
  __shared__ double s_total[N * N];
  __shared__ int s_token[N * N];  // -1: no offer
  __shared__ bool s_done[N];
  const int lane = threadIdx.x & (kWave - 1), b = threadIdx.x >> 6, group = blockIdx.x, row = group * p.beams + b;
  const double kNone = -(double)INFINITY;
  if (b < p.beams) {
    // Everything is asked for at once, also of a beam that has finished: what beam_rows_kernel left out is room of the workspace all the same.
    const float* ml = p.ml + (size_t)row * p.pieces * 2;
    const size_t at = (size_t)row * p.pieces * p.keep;
    const int n = p.pieces * p.keep;
    constexpr int E = 4;
    float val[E + 1];
    int id[E + 1];
    auto fetch = [&](int i0) {
#pragma unroll
      for (int i = 0; i < E; i++) {
        const int j = i0 + i * kWave + lane;
        const int k = p.ids[at + min(j, n - 1)];
        const float v = p.vals[at + min(j, n - 1)];
        id[i] = j < n ? k : -1;
        val[i] = id[i] >= 0 ? v : -INFINITY;
      }
    };
    const bool done = p.finished && p.finished[row];
    const float score = p.scores[row], m0 = ml[2 * min(lane, p.pieces - 1)], l0 = ml[2 * min(lane, p.pieces - 1) + 1];
    fetch(0);
    double total = kNone;
    int token = lane < p.V ? lane : -1;  // where nothing is finite, the lowest ones
    if (done) {
      if (fabsf(score) < INFINITY) {
        token = lane == 0 ? (int)p.eos : lane - 1 < p.eos ? lane - 1 : lane;  // behind eos what no finished beam does, at -infinity
        if (token >= p.V) token = -1;
        if (lane == 0) total = score;
      }
    } else {
      float m = m0;
      for (int i = lane + kWave; i < p.pieces; i += kWave) m = fmaxf(m, ml[2 * i]);
      m = wave_max(m);
      const float base = m == -INFINITY ? 0.f : m;
      double sum = 0.0;
      for (int i = lane; i < p.pieces; i += kWave) {
        const float mi = i == lane ? m0 : ml[2 * i], li = i == lane ? l0 : ml[2 * i + 1];
        sum += mi == -INFINITY ? (double)li : (double)li * exp((double)mi - base);
      }
#pragma unroll
      for (int o = 1; o < kWave; o <<= 1) sum += __shfl_xor(sum, o, kWave);
      const double lse = (double)base + log(sum);
      if (fabsf(score) < INFINITY && fabs(lse) < (double)INFINITY) {
        val[E] = -INFINITY;
        id[E] = -1;
        for (int i0 = 0; i0 < n; i0 += E * kWave) {
          if (i0) fetch(i0);
          wave_best<E + 1>(val, [&](int i) { return id[i]; }, p.keep, lane, s_list[b], s_best[b]);
          id[E] = lane < p.keep ? s_best[b].id[lane] : -1;
          val[E] = id[E] >= 0 ? s_best[b].val[lane] : -INFINITY;
        }
        token = id[E];
        const double x = (double)score + ((double)val[E] - lse);
        if (token >= 0 && fabs(x) < (double)INFINITY) total = x;
      }
    }
    if (lane < p.keep) {
      s_total[b * p.keep + lane] = total;
      s_token[b * p.keep + lane] = token;
    }
    if (lane == 0) s_done[b] = done;
  }
  __syncthreads();
  if (b != 0) return;
  const int n = p.beams * p.keep;
  constexpr int E = N * N / kWave;
  uint64_t key[E];
  float most = -INFINITY, near[E];
#pragma unroll
  for (int i = 0; i < E; i++) {
    const int c = i * kWave + lane;
    const bool in = c < n && s_token[c] >= 0;
    const double t = in ? s_total[c] : kNone;
    key[i] = in ? beam_key(t) : 0;
    near[i] = (float)t;
    most = fmaxf(most, near[i]);
  }
  const float bound = wave_kth(most, p.keep, lane);
  int count = 0;
  int* const list = s_list[0].id;
#pragma unroll
  for (int i = 0; i < E; i++) {
    const bool in = key[i] && near[i] >= bound;  // all of them where the bound is -infinity
    const uint64_t at = __ballot(in);
    const int j = count + ballot_rank(at);
    if (in && j < kWave) list[j] = i * kWave + lane;
    count += __popcll(at);
  }
  wave_lds_sync();
  auto give = [&](int c, int rank) {
    if (rank >= p.keep) return;
    const int out = group * p.keep + rank, parent = c / p.keep, token = s_token[c];
    p.scores_out[out] = (float)s_total[c];
    p.parents_out[out] = parent;
    p.tokens_out[out] = token;
    p.finished_out[out] = token == p.eos || s_done[parent];
  };
  if (count <= kWave) {
    const int c = lane < count ? list[lane] : 0;  // the list is in order
    const uint64_t mine = beam_key(s_total[c]);
    int rank = 0;
    for (int j = 0; j < count; j++) {
      const uint64_t other = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(mine >> 32), j) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)mine, j);
      rank += other > mine || (other == mine && j < lane);
    }
    if (lane < count) give(c, rank);
  } else {
#pragma unroll
    for (int i = 0; i < E; i++) {
      const int c = i * kWave + lane;
      int rank = 0;
      for (int j = 0; j < n; j++) {
        const uint64_t other = s_token[j] >= 0 ? beam_key(s_total[j]) : 0;
        rank += other > key[i] || (other == key[i] && j < c);
      }
      if (key[i]) give(c, rank);
    }
  }
}

// ---- reordering --------------------------------------------------------------------------------------------------------------------
// cache[g * beams + j] <- cache[g * beams + parent[g][j]] in place, for the entries that are live.  A thread takes one unit of 16 bytes (4 where a
// cache is not made of those) of all beams of a group: it asks for what moves, then stores it, so nothing is read behind a store.
// Every workgroup walks the live part of its caches, whatever room they have behind it.  Bound by memory: 32 rows of 4000 tokens in 8 bits, two layers of
// 8 heads of 128, 82 us, 4.9 TB/s, the rate of a copy.

struct ReorderCache {
  char* data;             // (groups * beams, heads, entries) of entry_bytes
  long long entry_bytes;
  int heads, entries;
  int slots;              // tokens an entry holds; 0: all entries are live
  int unit;               // 16 or 4
};
constexpr int kReorderCaches = 32;  // of a launch
struct ReorderArgs {
  ReorderCache c[kReorderCaches];
  const int64_t* parents;  // (groups, beams)
  const int64_t* lengths;  // tokens of a row
  int lengths_step, beams;
};

template <int N, class U>
__device__ __forceinline__ void reorder_units(const ReorderArgs& p, const ReorderCache& c) {
  const int group = blockIdx.z;
  int from[N];
  long long live[N], most = 0;  // units of a head that move to each beam
#pragma unroll
  for (int j = 0; j < N; j++) {
    from[j] = j;
    live[j] = 0;
    if (j < p.beams) {
      const long long f = p.parents[(size_t)group * p.beams + j];
      if (f >= 0 && f < p.beams && f != j) {  // a parent that is none leaves the beam as it is
        from[j] = (int)f;
        long long e = c.entries;
        if (c.slots) {
          const long long len = p.lengths[(size_t)(group * p.beams + f) * p.lengths_step];
          e = len <= 0 ? 0 : min(e, (len - 1) / c.slots + 1);
        }
        live[j] = e * c.entry_bytes / (long long)sizeof(U);
        most = max(most, live[j]);
      }
    }
  }
  if (most == 0) return;
  const long long pitch = c.entries * c.entry_bytes / (long long)sizeof(U);  // units of a head
  U* data = (U*)c.data + (size_t)group * p.beams * c.heads * pitch;
  const unsigned per = (unsigned)((most + 255) / 256), steps = per * c.heads;  // steps of 256 units
  for (unsigned i = blockIdx.x; i < steps; i += gridDim.x) {
    const unsigned head = i / per;
    const long long at = (long long)(i - head * per) * 256 + threadIdx.x;
    U* d = data + head * pitch + at;
    U x[N];
#pragma unroll
    for (int j = 0; j < N; j++)
      if (at < live[j]) x[j] = d[(size_t)from[j] * c.heads * pitch];
#pragma unroll
    for (int j = 0; j < N; j++)
      if (at < live[j]) d[(size_t)j * c.heads * pitch] = x[j];
  }
}

template <int N>
__global__ __launch_bounds__(256) void cache_reorder_kernel(ReorderArgs p) {
  const ReorderCache& c = p.c[blockIdx.y];
  if (c.unit == 16) reorder_units<N, u32x4>(p, c);
  else reorder_units<N, uint32_t>(p, c);
}

}  // namespace cats
