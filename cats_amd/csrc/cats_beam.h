// Beam search on the device: the best continuations of every group of beams, and the caches moved to the beams that go on.
#pragma once
#include "cats_device.h"

namespace cats {

constexpr int kBeamMax = 16;  // beams of a group, before and after

// ---- selection ---------------------------------------------------------------------------------------------------------------------
//   total(b, v) = score[b] + logit[b][v] - log(sum over v of exp(logit[b][v]));   the best `keep` of a group, ties to the lowest b * V + v
// A beam that has finished goes on only as (b, eos) with its score.  Totals that are not finite count as -infinity.
//
// beam_rows_kernel: one pass over the logits.  A wave holds 64 E of them in registers and leaves their maximum, the sum of exponentials and
// the best `keep`.  For those: the keep-th best of the lanes' best values bounds what can be among them, so what is not below it is
// gathered (some more than `keep`) and ranked by comparing each with all; only where ties make that more than 64 are the best taken one by
// one.  The workgroup's four waves are joined.  beam_join_kernel: a workgroup per group, a wave per beam joins its row's pieces in the same way, and
// the beams' candidates are ranked by their totals in 64 bits: the order has to be that of the sums, which differ in their last bits only.

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
  uint32_t* keys;         // [row][piece][keep]
  int* ids;
  int beams, V, keep, pieces;
};

// Floats ordered as unsigned integers; NaN as -infinity, -0 as 0.  0 is below them all.
__device__ __forceinline__ uint32_t beam_key(float x) {
  const uint32_t b = __float_as_uint(x != x ? -INFINITY : x + 0.f);
  return b >> 31 ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float beam_value(uint32_t k) { return __uint_as_float(k >> 31 ? k & 0x7fffffffu : ~k); }

template <int CTRL>
__device__ __forceinline__ uint32_t dpp_max(uint32_t v) {
  return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true));
}
// Largest over the 64 lanes, the same in all; the steps of wave_sum.
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
  v = dpp_max<0xB1>(v);
  v = dpp_max<0x4E>(v);
  v = dpp_max<0x141>(v);
  v = dpp_max<0x140>(v);
  const uint32_t a = __builtin_amdgcn_readlane((int)v, 0), b = __builtin_amdgcn_readlane((int)v, 16), c = __builtin_amdgcn_readlane((int)v, 32),
                 d = __builtin_amdgcn_readlane((int)v, 48);
  return max(max(a, b), max(c, d));
}

struct BeamList {  // in LDS, of a wave
  uint32_t key[kWave];
  int id[kWave];
};

// Writes the best `keep` of the wave's keys to `best`, in order, ids ascending among equal keys; 0 behind the last.  A key of 0 is no entry.
template <int E>
__device__ __forceinline__ void wave_best(uint32_t (&key)[E], const int (&id)[E], int keep, int lane, BeamList& list, BeamList& best) {
  uint32_t mine = 0;
#pragma unroll
  for (int i = 0; i < E; i++) mine = max(mine, key[i]);
  uint32_t bound = 0, rest = mine;
  for (int k = 0; k < keep; k++) {
    bound = wave_max(rest);
    const uint64_t at = __ballot(rest == bound);
    if (lane == (int)__builtin_ctzll(at)) rest = 0;
  }
  bound = max(bound, 1u);
  int count = 0;
#pragma unroll
  for (int i = 0; i < E; i++) {
    const bool in = key[i] >= bound;
    const uint64_t b = __ballot(in);
    const int at = count + ballot_rank(b);
    if (in && at < kWave) {
      list.key[at] = key[i];
      list.id[at] = id[i];
    }
    count += __popcll(b);
  }
  if (lane < keep) best.key[lane] = 0;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup", "local");
  __builtin_amdgcn_wave_barrier();
  if (count <= kWave) {
    const uint32_t k = lane < count ? list.key[lane] : 0u;
    const int v = lane < count ? list.id[lane] : INT32_MAX;
    int rank = 0;
    for (int j = 0; j < count; j++) {
      const uint32_t kj = __builtin_amdgcn_readlane((int)k, j);
      const int vj = __builtin_amdgcn_readlane(v, j);
      rank += kj > k || (kj == k && vj < v);
    }
    if (lane < count && rank < keep) {
      best.key[rank] = k;
      best.id[rank] = v;
    }
  } else {
    for (int k = 0; k < keep; k++) {
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < E; i++) top = max(top, key[i]);
      top = wave_max(top);
      uint32_t first = 0;  // of ids, turned round
#pragma unroll
      for (int i = 0; i < E; i++) first = key[i] == top ? max(first, ~(uint32_t)id[i]) : first;
      const int which = (int)~wave_max(first);
#pragma unroll
      for (int i = 0; i < E; i++) key[i] = id[i] == which ? 0u : key[i];
      if (lane == 0) {
        best.key[k] = top;
        best.id[k] = which;
      }
    }
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup", "local");
  __builtin_amdgcn_wave_barrier();
}

template <class DT, int E>
__global__ __launch_bounds__(256) void beam_rows_kernel(BeamArgs p) {
  typedef typename DT::st st;
  constexpr int VEC = DT::VEC, W = 4;
  __shared__ BeamList s_list[W], s_best[W];
  __shared__ float s_ml[W][2];
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x >> 6, row = blockIdx.y, piece = blockIdx.x;
  if (p.finished && p.finished[row]) return;
  const st* x = (const st*)p.logits + row * p.row_stride;
  const int first = (piece * W + wave) * kWave * E;  // the wave's elements, in vectors of VEC that go round the lanes
  uint32_t key[E];
  int id[E];
  float val[E];
  const bool whole = first + kWave * E <= p.V && ((uintptr_t)x & 15u) == 0;
#pragma unroll
  for (int i = 0; i < E / VEC; i++) {
    const int at = first + (i * kWave + lane) * VEC;
    if (whole) {
      const u32x4 w = load_stream((const u32x4*)(x + at));
#pragma unroll
      for (int e = 0; e < VEC; e++) {
        if constexpr (VEC == 4) val[i * VEC + e] = __uint_as_float(w[e]);
        else val[i * VEC + e] = DT::tof((st)(w[e / 2] >> (16 * (e & 1))));
      }
    } else {
#pragma unroll
      for (int e = 0; e < VEC; e++) val[i * VEC + e] = at + e < p.V ? DT::tof(x[at + e]) : 0.f;
    }
#pragma unroll
    for (int e = 0; e < VEC; e++) {
      id[i * VEC + e] = at + e;
      key[i * VEC + e] = at + e < p.V ? beam_key(val[i * VEC + e]) : 0u;
    }
  }
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < E; i++) top = max(top, key[i]);
  top = wave_max(top);
  const float m = top ? beam_value(top) : -INFINITY, base = m == -INFINITY ? 0.f : m;
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < E; i++) sum += key[i] ? expf(val[i] - base) : 0.f;
  sum = wave_sum(sum);
  wave_best<E>(key, id, p.keep, lane, s_list[wave], s_best[wave]);
  if (lane == 0) {
    s_ml[wave][0] = m;
    s_ml[wave][1] = sum;
  }
  __syncthreads();
  if (wave != 0) return;
  uint32_t k1[1] = {0};
  int i1[1] = {0};
  if (lane < W * p.keep) {
    k1[0] = s_best[lane / p.keep].key[lane % p.keep];
    i1[0] = s_best[lane / p.keep].id[lane % p.keep];
  }
  float mm = s_ml[0][0];
#pragma unroll
  for (int w = 1; w < W; w++) mm = fmaxf(mm, s_ml[w][0]);
  const float bb = mm == -INFINITY ? 0.f : mm;
  float ss = 0.f;
#pragma unroll
  for (int w = 0; w < W; w++) ss += s_ml[w][0] == -INFINITY ? s_ml[w][1] : s_ml[w][1] * expf(s_ml[w][0] - bb);
  __builtin_amdgcn_wave_barrier();
  wave_best<1>(k1, i1, p.keep, lane, s_list[0], s_best[0]);
  const size_t out = (size_t)row * p.pieces + piece;
  if (lane < p.keep) {
    p.keys[out * p.keep + lane] = s_best[0].key[lane];
    p.ids[out * p.keep + lane] = s_best[0].id[lane];
  }
  if (lane == 0) {
    p.ml[2 * out] = mm;
    p.ml[2 * out + 1] = ss;
  }
}

// Candidates of a row come in pieces of `keep`; a wave takes 64 at a time beside the best it has.
template <int N>
__global__ __launch_bounds__(N* kWave) void beam_join_kernel(BeamArgs p) {
  __shared__ BeamList s_list[N], s_best[N];
  __shared__ double s_total[N * N];
  __shared__ long long s_flat[N * N];
  const int lane = threadIdx.x & (kWave - 1), b = threadIdx.x >> 6, group = blockIdx.x, row = group * p.beams + b;
  const double kNone = -(double)INFINITY;
  if (b < p.beams) {
    const bool done = p.finished && p.finished[row];
    const float score = p.scores[row];
    double total = kNone;
    long long token = lane;  // where nothing is finite, the lowest ones
    if (done) {
      token = lane == 0 ? p.eos : lane - 1 < p.eos ? lane - 1 : lane;  // behind eos what no finished beam does, at -infinity
      if (token >= p.V) token = -1;
      if (lane == 0 && fabsf(score) < INFINITY) total = score;
    } else {
      const float* ml = p.ml + (size_t)row * p.pieces * 2;
      uint32_t top = 0;
      for (int i = lane; i < p.pieces; i += kWave) top = max(top, beam_key(ml[2 * i]));
      const float m = beam_value(wave_max(top)), base = m == -INFINITY ? 0.f : m;
      double sum = 0.0;
      for (int i = lane; i < p.pieces; i += kWave)
        sum += ml[2 * i] == -INFINITY ? (double)ml[2 * i + 1] : (double)ml[2 * i + 1] * exp((double)ml[2 * i] - base);
#pragma unroll
      for (int o = 1; o < kWave; o <<= 1) sum += __shfl_xor(sum, o, kWave);
      const double lse = (double)base + log(sum);
      const bool fine = fabsf(score) < INFINITY && fabs(lse) < (double)INFINITY;
      if (fine) {
        const size_t at = (size_t)row * p.pieces * p.keep;
        const int n = p.pieces * p.keep;
        uint32_t key[2] = {0, 0};
        int id[2] = {0, 0};
        for (int i0 = 0; i0 < n; i0 += kWave) {
          key[0] = i0 + lane < n ? p.keys[at + i0 + lane] : 0u;
          id[0] = key[0] ? p.ids[at + i0 + lane] : 0;
          const uint32_t have = key[1];
          if (i0 == 0 || wave_max(key[0]) >= wave_max(lane == p.keep - 1 ? have : 0u)) {
            wave_best<2>(key, id, p.keep, lane, s_list[b], s_best[b]);
            key[1] = lane < p.keep ? s_best[b].key[lane] : 0u;
            id[1] = key[1] ? s_best[b].id[lane] : 0;
          }
        }
        token = key[1] ? id[1] : -1;
        const double x = (double)score + ((double)beam_value(key[1]) - lse);
        if (key[1] && fabs(x) < (double)INFINITY) total = x;
      } else if (lane >= p.V) {
        token = -1;
      }
    }
    if (lane < p.keep) {
      s_total[b * p.keep + lane] = total;
      s_flat[b * p.keep + lane] = token < 0 ? -1 : (long long)b * p.V + token;
    }
  }
  __syncthreads();
  const int n = p.beams * p.keep;
  if (threadIdx.x >= n) return;
  const double mine = s_total[threadIdx.x];
  const long long flat = s_flat[threadIdx.x];
  if (flat < 0) return;
  int rank = 0;
  for (int j = 0; j < n; j++) rank += s_flat[j] >= 0 && (s_total[j] > mine || (s_total[j] == mine && s_flat[j] < flat));
  if (rank >= p.keep) return;
  const int out = group * p.keep + rank, parent = threadIdx.x / p.keep;
  const long long token = flat - (long long)parent * p.V;
  p.scores_out[out] = (float)mine;
  p.parents_out[out] = parent;
  p.tokens_out[out] = token;
  p.finished_out[out] = token == p.eos || (p.finished && p.finished[group * p.beams + parent]);
}

// ---- reordering --------------------------------------------------------------------------------------------------------------------
// cache[g * beams + j] <- cache[g * beams + parent[g][j]] in place, for the entries that are live.  A thread takes one unit of 16 bytes (4 where a
// cache is not made of those) of all beams of a group: it asks for what moves, then stores it, so nothing is read behind a store.
// Every workgroup walks the live part of its caches, whatever room they have behind it.  Bound by memory.

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
          e = len <= 0 ? 0 : min(e, (len + c.slots - 1) / c.slots);
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
